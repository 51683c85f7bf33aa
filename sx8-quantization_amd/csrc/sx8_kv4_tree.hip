// sx8_kv4_tree.hip -- attention of trees of drafted tokens over the paged 4-bit cache (include/sx8_paged.h).
//
// The products are those of sx8_kv4.hip: S^T = K Q^T with the levels as fp16 subnormals, O^T += V^T P^T with p * s as two
// fp16 numbers, the minima's parts in matrix products of their own, where a row of ones gives the weights' sum as well.  What
// differs is the shape of the work: a tree brings tens of query rows a KV head, so a unit is one or two tiles of 16 of them (a
// block's levels are unpacked once for both); a work-group's four waves take a unit's blocks in turn and add their results up in
// LDS, so that a unit cut over many work-groups leaves one partial result for each.  A block that ends at or behind the
// first new token is masked by 32 bits of each column's mask.
// Bound by instructions: for 16 rows and a block of 32 tokens of a head of 128 there are 28 matrix instructions of 16 cycles
// and 95 others of 4 (exponentials 16), beside 180 for the block; they take turns on a SIMD (two long trees: the VALU is busy 66%
// of its cycles, the matrix cores 33%, together 99%), and a second wave there makes neither faster.
// A wave keeps one block in registers: K of the next one is requested when the scores are done, V when the products are;
// no branch lies between (with one the sums are copied: 316 us for the two long trees below, at that stage 237).  Query fragments
// stay in LDS.  Three tiles a unit spill registers (245 us beside 198 on one machine), four leave one wave a SIMD (220).  With two
// (244 vector registers for heads of 128, two waves a SIMD; heads of 256 take 248 for one) no vector register is spilled, but 80 to 85 scalar
// ones lie in vector lanes (64 to 67 with one tile).
// Measured, with combine: 24 trees of 1 .. 24 rows after up to 8000 tokens, 32 heads over 8 of 128: 46 us; 8 of 64 rows after
// 2500 .. 4100: 84; two of 31 after 61000 and 100000, 32 over 4: 175 (under a profiler's clock 205).
#include "sx8_kv4_core.h"

namespace sx8 {
namespace {

// Record of a cut unit for the combine, at the work-group that has its first block; parts == 0: none.
struct TreePiece {
    int32_t parts, first, tile, head, row0, n, pad[2];      // first: place of its first part
};
static_assert(sizeof(TreePiece) == 32, "record");

struct TreeIo {
    const uint16_t* q;
    uint16_t* out;
    int64_t q_ts, q_hs, o_ts, o_hs;
    const uint64_t* mask;                 // [rows][words]
    int words;
    float scale_log2;
    float* part_o;                        // [2 groups][cols][HD]
    float* part_ml;                       // [2 groups][cols][2]
    TreePiece* piece;                     // [groups]
};

constexpr int kMaxWords = 4;              // of a row's mask: 256 drafted tokens a slot
// Work-groups a CU by tiles of 16 query rows, as registers allow.
template <int HD, int kCt>
constexpr int groups_per_cu() { return HD < 256 && kCt == 1 ? 3 : 2; }
constexpr int kMaxGroups = 768;
// Query rows of all partial results: the most that 256 groups_per_cu work-groups have, two units each.
constexpr int64_t part_rows(int64_t hd) { return hd == 256 ? 2 * 512 * 16 : 2 * 512 * 32; }
constexpr int64_t tree_ws(int64_t hd) { return part_rows(hd) * (hd + 2) * 4 + kMaxGroups * (int64_t)sizeof(TreePiece); }

__device__ __forceinline__ f32x4 zero4() { return f32x4{0.f, 0.f, 0.f, 0.f}; }

// x of eight values as two fp16 numbers each, hi + lo, both cut (rounded ones spill registers: 191 us beside 175 for two long trees)
__device__ __forceinline__ void halves8(const float* x, f16x8* hi, f16x8* lo) {
    typedef __fp16 h2 __attribute__((ext_vector_type(2)));
    u32x4 a, b;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const h2 h = __builtin_amdgcn_cvt_pkrtz(x[2 * i], x[2 * i + 1]);
        a[i] = __builtin_bit_cast(uint32_t, h);
        b[i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(__builtin_fmaf((float)h[0], -1.f, x[2 * i]), __builtin_fmaf((float)h[1], -1.f, x[2 * i + 1])));
    }
    *hi = __builtin_bit_cast(f16x8, a);
    *lo = __builtin_bit_cast(f16x8, b);
}
// (hi + lo) s of eight values as two fp16 numbers each: the product of the upper halves rounded, and what that left (the exact
// product of two fp16 numbers less its rounding is an fp16 number, down to the type's smallest) plus the lower halves'
// product: 12 instructions, 24 by products in float32 that are taken apart again (two long trees: 175 us, 191).
__device__ __forceinline__ void scaled8(f16x8 hi, f16x8 lo, f16x8 s, f16x8* a, f16x8* b) {
    *a = hi * s;
    *b = __builtin_elementwise_fma(lo, s, __builtin_elementwise_fma(hi, s, -*a));
}
template <int HD, bool kBf16, int kCt>
__global__ __launch_bounds__(256, (groups_per_cu<HD, kCt>())) void k_kv4_tree(const Kv4Pool p, const TreeIo io) {
    using Regs = Kv4Regs<HD>;
    constexpr int W = Regs::W, NT = Regs::NT, NG = Regs::NG, kBB = kv4_block_bytes(HD), kCols = 16 * kCt;
    constexpr float kInf = __builtin_inff();
    constexpr int kDims = 32, kPad = kDims + 4;                      // dimensions added up at a time
    __shared__ __align__(16) float sums[4][kCols][kPad];
    __shared__ __align__(16) u32x4 frag[kCt][W + 1][64];             // query fragments, and the sums of their groups
    __shared__ uint64_t masks[kCols][kMaxWords];
    __shared__ float unscale[kCols], ml[4][kCols][2];
    int64_t* const pre = reinterpret_cast<int64_t*>(dyn_lds);
    const int tid = threadIdx.x, lane = tid & 63, c = lane & 15, h = lane >> 4;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6), group = blockIdx.x;
    const int S = p.sh.n_slots, G = p.sh.G;
    auto places = [&](int s) {
        int first, n;
        kv4_rows(p.sh, p.cu, s, &first, &n);
        return kv4_tree_places(p.sh, kCols, n, kv4_len(p.sh, p.lens, s));
    };
    // the line: with up to 64 slots lane s holds the end of slot s, with more the ends lie in LDS
    const bool few = S <= 64;
    int64_t ends = 0, total;
    if (few) {
        ends = wave_prefix(lane < S ? places(lane) : 0);
        total = lane_of(ends, 63);
    } else {
        prefix_sums<256>(S, pre, places);
        __syncthreads();
        total = uniform(pre[S]);
    }
    const int64_t share = kv4_tree_share(total, gridDim.x);
    const int64_t x0 = group * share, x1 = x0 + share < total ? x0 + share : total;
    int slot = 0;
    if (x0 < total) {
        if (few) slot = __builtin_popcountll(__builtin_amdgcn_ballot_w64(lane < S && ends <= x0));
        else
            for (int s = lane; s - lane < S; s += 64)
                slot += __builtin_popcountll(__builtin_amdgcn_ballot_w64(s < S && pre[s < S ? s + 1 : S] <= x0));
    }
    if (tid == 0) io.piece[group].parts = 0;
    for (int64_t x = x0; x < x1;) {
        while (x >= (few ? lane_of(ends, slot) : uniform(pre[slot + 1]))) ++slot;
        const int64_t begin = few ? (slot ? lane_of(ends, slot - 1) : 0) : uniform(pre[slot]);
        int row0, n;
        kv4_rows(p.sh, p.cu, slot, &row0, &n);
        row0 = __builtin_amdgcn_readfirstlane(row0);
        n = __builtin_amdgcn_readfirstlane(n);
        const int len = __builtin_amdgcn_readfirstlane(kv4_len(p.sh, p.lens, slot));
        const int nb = kv4_unit_blocks(len), tiles = kv4_tree_tiles(n, G, kCols), first = len - n;
        const Kv4Run run = kv4_run(x, x - begin, x1, nb, kTreeBegin);
        const int b0 = run.b0, b1 = run.b1;
        const int64_t here = x;
        x += run.places;
        if (b0 == b1) continue;
        const int head = (int)kv4_div(run.unit, tiles), tile = (int)(run.unit - (int64_t)head * tiles);
        const int cols = min(kCols, n * G - kCols * tile);           // rows of the unit
        const int end = len > 0 ? b1 : b0;                           // (no token: no block)
        const int cnt = end > b0 + w ? (end - b0 - w + 3) / 4 : 0;   // blocks b0 + w, b0 + w + 4, ...
        int pages = -1;                                              // lane i: page of this wave's block i0 + i
        auto load_pages = [&](int i0) {
            const int b = b0 + w + 4 * (i0 + lane);
            pages = b < end ? p.table[(int64_t)slot * p.max_pages + (b >> p.bpp_log2)] : -1;
        };
        // where block i of the wave lies (a page that is none: its place in page 0, and bad)
        auto where = [&](int i, bool* bad) -> const uint8_t* {
            if (i != 0 && (i & 63) == 0) load_pages(i);
            const int b = b0 + w + 4 * i;
            const int page = __builtin_amdgcn_readlane(pages, i & 63);
            *bad = page < 0 || page >= p.n_pages;
            return p.pages + (*bad ? 0 : page) * p.page_bytes + (int64_t)((head << p.bpp_log2) + (b & ((1 << p.bpp_log2) - 1))) * kBB;
        };
        load_pages(0);
        __syncthreads();                                             // the last unit's LDS is free
        // query fragments: fp16 with each row's largest value in [64, 128); the groups' sums as two fp16 numbers
        for (int ct = w; ct < kCt; ct += 4) {
            const int r = kCols * tile + 16 * ct + c, tok = r / G;
            const bool row_ok = 16 * ct + c < cols;
            const uint16_t* qr = io.q + ((int64_t)row0 + (row_ok ? tok : 0)) * io.q_ts + (head * G + (row_ok ? r - tok * G : 0)) * io.q_hs + 8 * h;
            u32x4 raw[W];
            float top = 0.f;
#pragma unroll
            for (int j = 0; j < W; ++j) raw[j] = *reinterpret_cast<const u32x4*>(qr + 32 * j);
#pragma unroll
            for (int j = 0; j < W; ++j)
#pragma unroll
                for (int e = 0; e < 8; ++e) top = fmaxf(top, __builtin_fabsf(ld16<kBf16>(half_of(raw[j][e >> 1], e))));
            top = max4(row_ok ? top : 0.f);
            // exponent of the largest value; no scaling of rows that are zero or not finite
            const int ex = (int)(__builtin_bit_cast(uint32_t, top) >> 23);
            const int up = top > 0.f && ex < 255 && ex > 0 ? (127 + 6 - ex < 126 ? 127 + 6 - ex : 126) : 0;
            const float mul = __builtin_ldexpf(1.f, up);
            float qs[NG];
#pragma unroll
            for (int g = 0; g < NG; ++g) qs[g] = 0.f;
#pragma unroll
            for (int j = 0; j < W; ++j) {
                f16x8 f;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    f[e] = (_Float16)(row_ok ? ld16<kBf16>(half_of(raw[j][e >> 1], e)) * mul : 0.f);
                    qs[j / 2] += (float)f[e];
                }
                frag[ct][j][lane] = __builtin_bit_cast(u32x4, f);
            }
            f16x8 qm;
#pragma unroll
            for (int e = 0; e < 8; ++e) qm[e] = (_Float16)0.f;
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                const float s = sum4(qs[g]);
                const _Float16 hi = (_Float16)s;
                if (h == 0) {
                    qm[g] = hi;
                    qm[4 + g] = (_Float16)(s - (float)hi);
                }
            }
            frag[ct][W][lane] = __builtin_bit_cast(u32x4, qm);
            if (h == 0) unscale[16 * ct + c] = io.scale_log2 * __builtin_ldexpf(1.f, -up);
        }
        // masks: bits of rows that the slot has
        for (int i = tid; i < kCols * kMaxWords; i += 256) {
            const int col = i / kMaxWords, word = i % kMaxWords, left = n - 64 * word;
            uint64_t m = 0;
            if (col < cols && word < io.words && left > 0) {
                m = io.mask[((int64_t)row0 + (kCols * tile + col) / G) * io.words + word];
                if (left < 64) m &= (1ull << left) - 1ull;
            }
            masks[col][word] = m;
        }
        Regs rg;
        bool bad = false;
        if (cnt > 0) load_block<HD>(rg, where(0, &bad), lane);
        __syncthreads();
        float kscale[kCt], m[kCt];
        f32x4 o[kCt][NT], om[kCt];
#pragma unroll
        for (int ct = 0; ct < kCt; ++ct) {
            kscale[ct] = unscale[16 * ct + c];
            m[ct] = -kInf;
            om[ct] = zero4();
#pragma unroll
            for (int t = 0; t < NT; ++t) o[ct][t] = zero4();
        }
        for (int i = 0; i < cnt; ++i) {
            bool bad_next;
            const uint8_t* const next = where(i + 1 < cnt ? i + 1 : i, &bad_next);    // (the last block is loaded again)
            const int b = b0 + w + 4 * i;
            asm volatile("" ::: "memory");                           // (query fragments stay in LDS: registers)
            float pv[kCt][8];
#pragma unroll
            for (int a = 0; a < 2; ++a) {
                u32x4 mw = {0u, 0u, 0u, 0u};
                if (h == 0) {
                    mw.x = rg.km[a][0];
                    mw.z = rg.km[a][0];
                    if constexpr (NG == 4) mw.y = mw.w = rg.km[a][1];
                }
                f32x4 s[kCt];
#pragma unroll
                for (int ct = 0; ct < kCt; ++ct)
                    s[ct] = mfma16(__builtin_bit_cast(f16x8, mw), __builtin_bit_cast(f16x8, frag[ct][W][lane]), zero4());
#pragma unroll
                for (int g = 0; g < NG; ++g) {
                    const f16x8 l0 = levels(rg.kw[a][2 * g]), l1 = levels(rg.kw[a][2 * g + 1]);
                    float ks[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) ks[e] = sx8_h2f(half_of(rg.ks[g][2 * a + (e >> 1)], e)) * 1048576.f;
                    f32x4 acc[kCt];
#pragma unroll
                    for (int ct = 0; ct < kCt; ++ct) acc[ct] = mfma16(l0, __builtin_bit_cast(f16x8, frag[ct][2 * g][lane]), zero4());
#pragma unroll
                    for (int ct = 0; ct < kCt; ++ct) acc[ct] = mfma16(l1, __builtin_bit_cast(f16x8, frag[ct][2 * g + 1][lane]), acc[ct]);
#pragma unroll
                    for (int ct = 0; ct < kCt; ++ct)
#pragma unroll
                        for (int e = 0; e < 4; ++e) s[ct][e] = __builtin_fmaf(ks[e], acc[ct][e], s[ct][e]);
                }
#pragma unroll
                for (int ct = 0; ct < kCt; ++ct)
#pragma unroll
                    for (int e = 0; e < 4; ++e) pv[ct][4 * a + e] = s[ct][e];
            }
            load_block_k<HD>(rg, next, lane);
            u32x4 vm = rg.vm;
            if (b * 32 + 31 >= first || bad) {
                asm volatile("");                // (a branch: as selects these would run for every block)
#pragma unroll
                for (int ct = 0; ct < kCt; ++ct) {
                    const uint32_t see = bad ? 0u : kv4_tree_bits(masks[16 * ct + c], kMaxWords, first, b * 32) >> 4 * h;
#pragma unroll
                    for (int e = 0; e < 8; ++e) pv[ct][e] = see >> (e / 4 * 16 + e % 4) & 1u ? pv[ct][e] : -kInf;
                }
                // A token whose V is no number must not reach a column that may not attend it through 0 * NaN: its scale and
                // minimum (each may be one, in bytes that no token was written to) become zeros, and the columns that attend it
                // get the NaN by themselves, however small its weight.
                uint32_t nan[NG], any = 0, low = 0;                   // low: of lane c the minima of group c
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if ((half_of(vm[e >> 1], e) & 0x7FFFu) >= 0x7C00u) low |= 1u << (e / 4 * 16 + e % 4);
                any = low;
#pragma unroll
                for (int g = 0; g < NG; ++g) {
                    nan[g] = 0;
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        if ((half_of(rg.vs[g][e >> 1], e) & 0x7FFFu) >= 0x7C00u) nan[g] |= 1u << (e / 4 * 16 + e % 4);
                    any |= nan[g];
                }
                if (__builtin_amdgcn_ballot_w64(any != 0) != 0) {
#pragma unroll
                    for (int g = 0; g < NG; ++g) {
#pragma unroll
                        for (int e = 0; e < 8; ++e)
                            if (nan[g] >> (e / 4 * 16 + e % 4) & 1u) rg.vs[g][e >> 1] &= e & 1 ? 0xFFFFu : 0xFFFF0000u;
                        nan[g] = (nan[g] | __shfl((int)low, 16 * h + g, 64)) << 4 * h;
                        nan[g] |= __shfl_xor((int)nan[g], 16, 64);
                        nan[g] |= __shfl_xor((int)nan[g], 32, 64);
#pragma unroll
                        for (int ct = 0; ct < kCt; ++ct)
                            if (!bad && (kv4_tree_bits(masks[16 * ct + c], kMaxWords, first, b * 32) & nan[g]))
#pragma unroll
                                for (int t = 4 * g; t < 4 * g + 4; ++t) o[ct][t] += __builtin_nanf("");
                    }
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const uint32_t lo = vm[e] & 0x7FFFu, hi = vm[e] >> 16 & 0x7FFFu;
                        vm[e] = (lo >= 0x7C00u ? 0u : vm[e] & 0xFFFFu) | (hi >= 0x7C00u ? 0u : vm[e] & 0xFFFF0000u);
                    }
                }
            }
            float mx[kCt];
            bool over = false;
#pragma unroll
            for (int ct = 0; ct < kCt; ++ct) {
                mx[ct] = pv[ct][0];
#pragma unroll
                for (int e = 1; e < 8; ++e) mx[ct] = fmaxf(mx[ct], pv[ct][e]);
                mx[ct] *= kscale[ct];
                over |= mx[ct] > m[ct] + (kUp + kSlack);
            }
            if (__builtin_amdgcn_ballot_w64(over) != 0) {
#pragma unroll
                for (int ct = 0; ct < kCt; ++ct) {
                    const float mn = fmaxf(m[ct], max4(mx[ct] - kUp));
                    const float alpha = m[ct] == mn ? 1.f : __builtin_amdgcn_exp2f(m[ct] - mn);
                    m[ct] = mn;
                    om[ct] *= alpha;
#pragma unroll
                    for (int t = 0; t < NT; ++t) o[ct][t] *= alpha;
                }
            }
#pragma unroll
            for (int ct = 0; ct < kCt; ++ct) {
                const float nm = m[ct] == -kInf ? 0.f : -m[ct];
#pragma unroll
                for (int e = 0; e < 8; ++e) pv[ct][e] = __builtin_amdgcn_exp2f(__builtin_fmaf(pv[ct][e], kscale[ct], nm));
            }
            // rows of the minima's product: a group's minima, and behind them ones, whose sum is the weights'
            constexpr uint32_t kOnes = 0x3C003C00u;
            if (c == NG) vm = u32x4{kOnes, kOnes, kOnes, kOnes};
            if (c > NG) vm = u32x4{0u, 0u, 0u, 0u};
            const f16x8 vm8 = __builtin_bit_cast(f16x8, vm);
            f16x8 ph[kCt], pl[kCt];
#pragma unroll
            for (int ct = 0; ct < kCt; ++ct) {
                halves8(pv[ct], &ph[ct], &pl[ct]);
                om[ct] = mfma16(vm8, ph[ct], om[ct]);
                om[ct] = mfma16(vm8, pl[ct], om[ct]);
            }
            uint32_t large = 0;                  // bits 14 and 30: a scale of 2 or more (or NaN)
#pragma unroll
            for (int g = 0; g < NG; ++g) large |= rg.vs[g][0] | rg.vs[g][1] | rg.vs[g][2] | rg.vs[g][3];
            if (__builtin_amdgcn_ballot_w64((large & 0x40004000u) != 0) != 0) {
#pragma unroll
                for (int g = 0; g < NG; ++g) {
#pragma unroll 1
                    for (int k = 5; k <= 15; k += 5) {
                        u32x4 s = large_scales(rg.vs[g], k);
                        if (__builtin_amdgcn_ballot_w64((s[0] | s[1] | s[2] | s[3]) != 0) == 0) continue;
                        const _Float16 down = (_Float16)__builtin_ldexpf(1.f, -k), up = (_Float16)__builtin_ldexpf(1.f, k);
                        s = __builtin_bit_cast(u32x4, __builtin_bit_cast(f16x8, s) * f16x8(down));
#pragma unroll
                        for (int ct = 0; ct < kCt; ++ct) {
                            f16x8 hi, lo;
                            scaled8(ph[ct], pl[ct], __builtin_bit_cast(f16x8, s), &hi, &lo);
#pragma unroll
                            for (int t = 4 * g; t < 4 * g + 4; ++t) {
                                uint32_t word = rg.vw[t];
                                asm volatile("" : "+v"(word));          // (here, not ahead of the loop: registers)
                                const f16x8 lv = levels(word) * f16x8(up);
                                o[ct][t] = mfma16(lv, hi, o[ct][t]);
                                o[ct][t] = mfma16(lv, lo, o[ct][t]);
                            }
                        }
                    }
#pragma unroll
                    for (int e = 0; e < 4; ++e) rg.vs[g][e] &= ~((rg.vs[g][e] >> 14 & 0x00010001u) * 0xFFFFu);
                }
            }
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                f16x8 lv[4];
#pragma unroll
                for (int t = 0; t < 4; ++t) lv[t] = levels(rg.vw[4 * g + t]);
#pragma unroll
                for (int ct = 0; ct < kCt; ++ct) {
                    f16x8 hi, lo;
                    scaled8(ph[ct], pl[ct], __builtin_bit_cast(f16x8, rg.vs[g]), &hi, &lo);
#pragma unroll
                    for (int t = 0; t < 4; ++t) o[ct][4 * g + t] = mfma16(lv[t], hi, o[ct][4 * g + t]);
#pragma unroll
                    for (int t = 0; t < 4; ++t) o[ct][4 * g + t] = mfma16(lv[t], lo, o[ct][4 * g + t]);
                }
            }
            load_block_v<HD>(rg, next, lane);
            bad = bad_next;
        }
        // O = 2^20 (levels) + (the minima's sum of the group, row g of om); the weights' sum in row NG
        float l[kCt];
#pragma unroll
        for (int ct = 0; ct < kCt; ++ct) {
            l[ct] = __shfl(om[ct][NG % 4], c + 16 * (NG / 4), 64);
            if (h == 0) {
                ml[w][16 * ct + c][0] = m[ct];
                ml[w][16 * ct + c][1] = l[ct];
            }
        }
        __syncthreads();
        const bool whole = b0 == 0 && b1 == nb;
        float f[kCt];
#pragma unroll
        for (int ct = 0; ct < kCt; ++ct) {
            const int col = 16 * ct + c;
            const float mm = fmaxf(fmaxf(ml[0][col][0], ml[1][col][0]), fmaxf(ml[2][col][0], ml[3][col][0]));
            f[ct] = m[ct] == mm ? 1.f : __builtin_amdgcn_exp2f(m[ct] - mm);
            if (whole) {
                float sum = 0.f;
#pragma unroll
                for (int i = 0; i < 4; ++i) sum += ml[i][col][1] * (ml[i][col][0] == mm ? 1.f : __builtin_amdgcn_exp2f(ml[i][col][0] - mm));
                f[ct] *= sum == 0.f ? 0.f : 1.f / sum;
            }
        }
        const int place = 2 * group + (here == x0 ? 0 : 1);
        float* const po = io.part_o + (int64_t)place * kCols * HD;
#pragma unroll
        for (int d0 = 0; d0 < HD; d0 += kDims) {
            if (d0) __syncthreads();
#pragma unroll
            for (int ct = 0; ct < kCt; ++ct)
#pragma unroll
                for (int t = d0 / 16; t < d0 / 16 + kDims / 16; ++t) {
                    const float og = __shfl(om[ct][t / 4], c, 64);
                    f32x4 v;
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[e] = __builtin_fmaf(o[ct][t][e], 1048576.f, og) * f[ct];
                    *reinterpret_cast<f32x4*>(&sums[w][16 * ct + c][(t * 16 - d0) + 4 * h]) = v;
                }
            __syncthreads();
            for (int i = tid; i < kCols * (kDims / 4); i += 256) {
                const int col = i / (kDims / 4), d = i % (kDims / 4) * 4;
                if (col >= cols) break;
                f32x4 v = *reinterpret_cast<const f32x4*>(&sums[0][col][d]);
#pragma unroll
                for (int k = 1; k < 4; ++k) v += *reinterpret_cast<const f32x4*>(&sums[k][col][d]);
                if (whole) {
                    const int r = kCols * tile + col, tok = r / G;
                    *reinterpret_cast<u32x2*>(io.out + ((int64_t)row0 + tok) * io.o_ts + (head * G + (r - tok * G)) * io.o_hs + d0 + d) =
                        u32x2{pack16<kBf16>(v[0], v[1]), pack16<kBf16>(v[2], v[3])};
                } else {
                    *reinterpret_cast<f32x4*>(po + (int64_t)col * HD + d0 + d) = v;
                }
            }
        }
        if (!whole) {
            if (tid < cols) {
                const float mm = fmaxf(fmaxf(ml[0][tid][0], ml[1][tid][0]), fmaxf(ml[2][tid][0], ml[3][tid][0]));
                float sum = 0.f;
#pragma unroll
                for (int i = 0; i < 4; ++i) sum += ml[i][tid][1] * (ml[i][tid][0] == mm ? 1.f : __builtin_amdgcn_exp2f(ml[i][tid][0] - mm));
                io.part_ml[((int64_t)place * kCols + tid) * 2] = mm;
                io.part_ml[((int64_t)place * kCols + tid) * 2 + 1] = sum;
            }
            if (b0 == 0 && tid == 0) {
                TreePiece pc;
                pc.parts = (int)((begin + run.unit * (nb + kTreeBegin) + kTreeBegin + nb - 1) / share - group + 1);
                pc.first = place;
                pc.tile = tile;
                pc.head = head;
                pc.row0 = row0;
                pc.n = n;
                io.piece[group] = pc;
            }
        }
    }
}

// Units that were cut: wave (record, row) adds a row's parts up (part 0 at its place, part j at place 2 (group + j)), 64 of them at
// a time: each lane weighs one, and the sums are added in the parts' order, 16 requested together (96 parts: 6.2 us, 13.9 where
// every lane computes every weight).
template <int HD, bool kBf16, int kCols>
__global__ __launch_bounds__(256) void k_kv4_tree_combine(const TreeIo io, int G) {
    constexpr int N = HD / 64;
    typedef float vecN __attribute__((ext_vector_type(N)));
    const TreePiece pc = io.piece[blockIdx.x];
    const int row = blockIdx.y * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    if (pc.parts == 0 || row >= min(kCols, pc.n * G - kCols * pc.tile)) return;
    auto at = [&](int i) { return (int64_t)(i == 0 ? pc.first : 2 * (pc.first / 2 + i)) * kCols + row; };
    float m = -__builtin_inff(), den = 0.f;
    vecN acc = 0.f;
    for (int i0 = 0; i0 < pc.parts; i0 += 64) {                   // lane j: what part i0 + j weighs
        const int n = min(64, pc.parts - i0);
        const int64_t mine = at(i0 + min(lane, n - 1)) * 2;
        const float pm = io.part_ml[mine], pl = io.part_ml[mine + 1];
        float f = 0.f;
        // kU parts requested together
        auto add = [&](auto together, int i) {
            constexpr int kU = decltype(together)::value;
            vecN v[kU];
#pragma unroll
            for (int u = 0; u < kU; ++u) v[u] = reinterpret_cast<const vecN*>(io.part_o + at(i0 + min(i + u, n - 1)) * HD)[lane];
            __builtin_amdgcn_sched_barrier(0);
            if (i == 0) {
                float mn = fmaxf(m, pm);
#pragma unroll
                for (int o = 32; o > 0; o >>= 1) mn = fmaxf(mn, __shfl_xor(mn, o, 64));
                const float alpha = m == mn ? 1.f : __builtin_amdgcn_exp2f(m - mn);
                f = lane >= n ? 0.f : pm == mn ? 1.f : __builtin_amdgcn_exp2f(pm - mn);
                float sum = lane < n ? f * pl : 0.f;
#pragma unroll
                for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o, 64);
                m = mn;
                den = __builtin_fmaf(den, alpha, sum);
                acc *= alpha;
            }
#pragma unroll
            for (int u = 0; u < kU; ++u) {
                if (i + u >= n) continue;
                acc = __builtin_elementwise_fma(vecN(__builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, f), i + u))), v[u], acc);
            }
        };
        if (n <= 8) add(std::integral_constant<int, 8>{}, 0);
        else
            for (int i = 0; i < n; i += 16) add(std::integral_constant<int, 16>{}, i);
    }
    acc *= den == 0.f ? 0.f : 1.f / den;
    const int r = kCols * pc.tile + row, tok = r / G;
    uint16_t* dst = io.out + ((int64_t)pc.row0 + tok) * io.o_ts + (pc.head * G + (r - tok * G)) * io.o_hs + N * lane;
    if constexpr (N == 1) *dst = (uint16_t)st16<kBf16>(acc[0]);
    else
#pragma unroll
        for (int e = 0; e < N; e += 2) *reinterpret_cast<uint32_t*>(dst + e) = pack16<kBf16>(acc[e], acc[e + 1]);
}

}  // namespace
}  // namespace sx8

extern "C" int64_t sx8_kv4_attend_tree_workspace_bytes(int32_t hd) { return sx8::hd_ok(hd) ? sx8::tree_ws(hd) : -1; }

extern "C" int32_t sx8_kv4_attend_tree(const uint8_t* pages, const int32_t* table, const int32_t* lens, const int32_t* cu,
                                       int64_t n_slots, int64_t max_pages, int64_t n_pages, const void* q, void* out,
                                       int64_t rows, int64_t q_ts, int64_t q_hs, int64_t o_ts, int64_t o_hs,
                                       const uint64_t* mask, int32_t words, int32_t nh, int32_t nk, int32_t hd,
                                       int32_t page_tokens, float scale, int32_t dtype, void* workspace,
                                       int64_t workspace_bytes, void* stream) {
    using namespace sx8;
    const char* what = "sx8_kv4_attend_tree";
    Kv4Pool p;
    int32_t rc = make_pool(what, &p, pages, table, lens, cu, n_slots, max_pages, n_pages, rows, nk, hd, page_tokens, dtype);
    if (rc == SX8_OK) rc = check_rows(what, "q", q, q_ts, q_hs, rows);
    if (rc == SX8_OK) rc = check_rows(what, "out", out, o_ts, o_hs, rows);
    if (rc != SX8_OK) return rc;
    if (nh <= 0 || nh % nk || nh / nk > 256)
        return fail(SX8_ERR_INVALID, "%s: nh must be a multiple of nk, at most 256 nk", what);
    rc = check_apart(what, "out", o_ts, o_hs, rows, nh, hd);
    if (rc != SX8_OK) return rc;
    if (!(scale > 0.f) || !(scale < __builtin_inff()))
        return fail(SX8_ERR_INVALID, "%s: scale must be positive and finite", what);
    if ((!mask && rows > 0) || !aligned(mask, 8) || words < 1 || words > kMaxWords)
        return fail(SX8_ERR_INVALID, "%s: mask must be 8-byte aligned, of 1..%d words a row", what, kMaxWords);
    if (!workspace || workspace_bytes < tree_ws(hd) || !aligned(workspace, 256))
        return fail(SX8_ERR_INVALID, "%s: workspace needs %lld bytes, 256-byte aligned", what, (long long)tree_ws(hd));
    if (out == q && rows > 0) return fail(SX8_ERR_INVALID, "%s: out may not be q", what);
    if (rows * (nh / nk) > 0x7FFFFF00) return fail(SX8_ERR_UNSUPPORTED, "%s: over 2^31 query rows of a KV head", what);
    if (rows == 0) return ok();
    p.sh.G = nh / nk;
    TreeIo io{(const uint16_t*)q, (uint16_t*)out, q_ts, q_hs, o_ts, o_hs, mask, words, scale * 1.4426950408889634f, nullptr,
              nullptr, nullptr};
    io.piece = reinterpret_cast<TreePiece*>(workspace);
    io.part_o = reinterpret_cast<float*>(io.piece + kMaxGroups);
    io.part_ml = io.part_o + part_rows(hd) * hd;
    // tiles of 16 query rows that a slot has on the average
    const int64_t tiles = (rows * p.sh.G + 16 * n_slots - 1) / (16 * n_slots);
    by_kind(hd, dtype, [&](auto d, auto b) {
        constexpr int HD = decltype(d)::value;
        constexpr bool kBf = decltype(b)::value;
        auto go = [&](auto ct) {
            constexpr int kCt = decltype(ct)::value;
            constexpr unsigned groups = 256 * groups_per_cu<HD, kCt>();
            static_assert(groups <= kMaxGroups && 2 * groups * 16 * kCt <= part_rows(HD), "workspace");
            hipLaunchKernelGGL((k_kv4_tree<HD, kBf, kCt>), dim3(groups), dim3(256), n_slots <= 64 ? 0 : prefix_bytes(p),
                               as_stream(stream), p, io);
            const int64_t most = rows * p.sh.G < 16 * kCt ? rows * p.sh.G : 16 * kCt;
            hipLaunchKernelGGL((k_kv4_tree_combine<HD, kBf, 16 * kCt>), dim3(groups, (unsigned)(most + 3) / 4), dim3(256), 0,
                               as_stream(stream), io, p.sh.G);
        };
        // Two tiles a unit from four tiles a slot on, where registers allow it (8 slots of about 3300 tokens, 8 KV heads of 128,
        // groups of 4: 64 new rows 92 us instead of 108, 16 rows 37 instead of 40, 12 rows 36 instead of 34, 2 rows 27 instead of 23).
        if constexpr (HD < 256) {
            if (tiles >= 4) return go(std::integral_constant<int, 2>{});
        }
        go(std::integral_constant<int, 1>{});
    });
    return check_launch(what);
}
