// sx8_kv4.hip -- the paged 4-bit KV cache: writer, reader and attention (include/sx8_paged.h).
#include <type_traits>

#include "sx8_host.h"
#include "sx8_kv4_dev.h"
#include "sx8_paged.h"

namespace sx8 {
namespace {

// What every kernel over the slots gets.
struct Kv4Pool {
    const uint8_t* pages;
    const int32_t* table;
    const int32_t* lens;
    const int32_t* cu;
    int64_t page_bytes;
    int max_pages, n_pages, bpp_log2;      // blocks of a page: 1 << bpp_log2
    Kv4Shape sh;
};

// Byte offset of block b of head h of a slot's page, or -1 where the slot has no such page.
__device__ __forceinline__ int64_t block_offset(const Kv4Pool& p, int slot, int head, int64_t b, int bb) {
    const int64_t at = b >> p.bpp_log2;
    if (at >= p.max_pages) return -1;
    const int page = p.table[(int64_t)slot * p.max_pages + at];
    if (page < 0 || page >= p.n_pages) return -1;
    return page * p.page_bytes + (((int64_t)head << p.bpp_log2) + (b & ((1 << p.bpp_log2) - 1))) * bb;
}

// ---- append ------------------------------------------------------------------------------------
// A work-group encodes the new rows of one block of one head, so that no word of the cache has two writers.
// Eight lanes hold a group of 64 values (16 bytes each): minimum and maximum by three lane exchanges, then each
// lane's eight levels.  The level is decided in binary64, where x - m is exact for fp16 rows and the quotient is put
// right by its exact remainder, so that ties fall as the definition says.  K's eight levels of a lane are one
// word; V's word holds eight tokens of a dimension, so V's levels meet in LDS, and a word with tokens of
// earlier calls keeps their bits.
struct Enc {
    float s, m;
    uint32_t lv[8];
};

// rows outside the call come as zeros (their results are unused)
__device__ __forceinline__ void encode_group(const float (&x)[8], Enc& e) {
#pragma clang fp contract(off)
    float lo = x[0], hi = x[0];
    bool bad = false;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        lo = fminf(lo, x[i]);
        hi = fmaxf(hi, x[i]);
        bad |= !(__builtin_fabsf(x[i]) < __builtin_inff());
    }
    int b = bad;
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) {
        lo = fminf(lo, __shfl_xor(lo, o, 8));
        hi = fmaxf(hi, __shfl_xor(hi, o, 8));
        b |= __shfl_xor(b, o, 8);
    }
    const float r = hi - lo;
    e.s = (float)(_Float16)fminf(r * (1.0f / 15.0f), 65504.0f);
    e.m = (float)(_Float16)fminf(fmaxf(lo, -65504.0f), 65504.0f);
    if (b) e.s = e.m = __builtin_nanf("");
    const double s = e.s, m = e.m, inv = 1.0 / s;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const double d = (double)x[i] - m;
        double n = __builtin_rint(d * inv);
        n = n < 0.0 ? 0.0 : n > 15.0 ? 15.0 : n;
        // remainder d - n s (exact: n s has 15 bits); one step further where it is over half a step, or half and n odd
        const double rem = d - n * s;
        const bool odd = (int)n & 1;
        if (n < 15.0 && (2.0 * rem > s || (2.0 * rem == s && odd))) n += 1.0;
        else if (n > 0.0 && (-2.0 * rem > s || (-2.0 * rem == s && odd))) n -= 1.0;
        e.lv[i] = !b && s > 0.0 ? (uint32_t)(int)n : 0u;
    }
}

// The block that work item `item` of the call names: slot, its block, and the new tokens in it (block-relative
// [t0, t1), row of token t0).  Every thread gets it; false past the last item.
struct Touched {
    int slot;
    int64_t block;
    int t0, t1;
    int64_t row0;
};
__device__ __forceinline__ bool find_touched(const Kv4Pool& p, int64_t item, int64_t* pre, Touched* t) {
    prefix_sums<256>(p.sh.n_slots, pre, [&](int s) {
        int64_t first, n, b;
        kv4_rows(p.sh, p.cu, s, &first, &n);
        return kv4_touched(kv4_len(p.sh, p.lens, s), n, &b);
    });
    __syncthreads();
    if (item >= pre[p.sh.n_slots]) return false;
    t->slot = find_item<256>(p.sh.n_slots, pre, item);
    int64_t first, n, b;
    kv4_rows(p.sh, p.cu, t->slot, &first, &n);
    const int64_t len = kv4_len(p.sh, p.lens, t->slot);
    kv4_touched(len, n, &b);
    t->block = b + (item - pre[t->slot]);
    const int64_t a = len - n > t->block * 32 ? len - n : t->block * 32;
    const int64_t e = len < t->block * 32 + 32 ? len : t->block * 32 + 32;
    t->t0 = (int)(a - t->block * 32);
    t->t1 = (int)(e - t->block * 32);
    t->row0 = first + a - (len - n);
    return true;
}

struct RowsIn {
    const uint16_t* k;
    const uint16_t* v;
    int64_t k_ts, k_hs, v_ts, v_hs;
};

extern __shared__ __align__(16) unsigned char dyn_lds[];

template <int HD, bool kBf16>
__global__ __launch_bounds__(256) void k_kv4_append(const Kv4Pool p, const RowsIn in) {
    constexpr int kBB = kv4_block_bytes(HD), CPR = HD / 8;
    __shared__ uint8_t lv[32][HD + 4];
    int64_t* const pre = reinterpret_cast<int64_t*>(dyn_lds);
    Touched t;
    if (!find_touched(p, blockIdx.x, pre, &t)) return;
    const int head = blockIdx.y, tid = threadIdx.x;
    const int64_t off = block_offset(p, t.slot, head, t.block, kBB);
    if (off < 0) return;                                            // (uniform)
    uint8_t* const blk = const_cast<uint8_t*>(p.pages) + off;
    const int nt = t.t1 - t.t0;
    for (int which = 0; which < 2; ++which) {
        const uint16_t* src = which ? in.v : in.k;
        const int64_t ts = which ? in.v_ts : in.k_ts, hs = which ? in.v_hs : in.k_hs;
        // (whole groups of eight lanes run together: CPR is a multiple of 8)
        for (int i = tid; i < nt * CPR; i += 256) {
            const int tok = t.t0 + i / CPR, d0 = i % CPR * 8, g = d0 / kKv4Group;
            const u32x4 w = *reinterpret_cast<const u32x4*>(src + (t.row0 + i / CPR) * ts + head * hs + d0);
            float x[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = ld16<kBf16>(half_of(w[e >> 1], e));
            Enc en;
            encode_group(x, en);
            if (which == 0) {
                uint32_t word = 0;
#pragma unroll
                for (int e = 0; e < 8; ++e) word |= en.lv[e] << kv4_shift(e);
                *reinterpret_cast<uint32_t*>(blk + kv4_k_word(HD, tok, d0)) = word;
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) lv[tok][d0 + e] = (uint8_t)en.lv[e];
            }
            if (i % 8 == 0) {
                *reinterpret_cast<uint16_t*>(blk + kv4_param(HD, 2 * which, tok, g)) = (uint16_t)st16<false>(en.s);
                *reinterpret_cast<uint16_t*>(blk + kv4_param(HD, 2 * which + 1, tok, g)) = (uint16_t)st16<false>(en.m);
            }
        }
    }
    __syncthreads();
    for (int i = tid; i < HD * 4; i += 256) {
        const int d = i % HD, h = i / HD;                           // word: tokens 4 h + r and 16 + 4 h + r
        uint32_t word = 0, fresh = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const int tok = e / 4 * 16 + 4 * h + e % 4;
            if (tok >= t.t0 && tok < t.t1) {
                word |= (uint32_t)lv[tok][d] << kv4_shift(e);
                fresh |= 15u << kv4_shift(e);
            }
        }
        if (fresh == 0) continue;
        uint32_t* const at = reinterpret_cast<uint32_t*>(blk + kv4_v_word(HD, 4 * h, d));
        *at = fresh == 0xFFFFFFFFu ? word : (*at & ~fresh) | word;
    }
}

// ---- read --------------------------------------------------------------------------------------
// The same cut: a work-group takes one block of one head into LDS (coalesced) and writes its new tokens' rows.
struct RowsOut {
    uint16_t* k;
    uint16_t* v;
    int64_t k_ts, k_hs, v_ts, v_hs;
};

template <int HD, bool kBf16>
__global__ __launch_bounds__(256) void k_kv4_read(const Kv4Pool p, const RowsOut out) {
    constexpr int kBB = kv4_block_bytes(HD), CPR = HD / 8;
    __shared__ __align__(16) uint8_t blk[kBB];
    int64_t* const pre = reinterpret_cast<int64_t*>(dyn_lds);
    Touched t;
    if (!find_touched(p, blockIdx.x, pre, &t)) return;
    const int head = blockIdx.y, tid = threadIdx.x;
    const int64_t off = block_offset(p, t.slot, head, t.block, kBB);
    if (off < 0) return;                                            // (uniform)
    for (int i = tid; i < kBB / 16; i += 256)
        reinterpret_cast<u32x4*>(blk)[i] = reinterpret_cast<const u32x4*>(p.pages + off)[i];
    __syncthreads();
    const int nt = t.t1 - t.t0;
    for (int i = tid; i < 2 * nt * CPR; i += 256) {
        const int which = i >= nt * CPR, j = i - which * nt * CPR;
        const int tok = t.t0 + j / CPR, d0 = j % CPR * 8, g = d0 / kKv4Group;
        const float s = sx8_h2f(*reinterpret_cast<const uint16_t*>(blk + kv4_param(HD, 2 * which, tok, g)));
        const float m = sx8_h2f(*reinterpret_cast<const uint16_t*>(blk + kv4_param(HD, 2 * which + 1, tok, g)));
        const uint32_t kw = *reinterpret_cast<const uint32_t*>(blk + kv4_k_word(HD, tok, d0));
        u32x4 w;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const uint32_t vw = *reinterpret_cast<const uint32_t*>(blk + kv4_v_word(HD, tok, d0 + e));
            const uint32_t l = which ? (vw >> kv4_v_shift(tok)) & 15u : (kw >> kv4_shift(e)) & 15u;
            const uint32_t b = st16<kBf16>(__builtin_fmaf((float)(int)l, s, m));
            if (e & 1) w[e >> 1] |= b << 16;
            else w[e >> 1] = b;
        }
        uint16_t* const dst = which ? out.v + (t.row0 + j / CPR) * out.v_ts + head * out.v_hs
                                    : out.k + (t.row0 + j / CPR) * out.k_ts + head * out.k_hs;
        *reinterpret_cast<u32x4*>(dst + d0) = w;
    }
}

// ---- attend ------------------------------------------------------------------------------------
// Work-groups share the blocks of all units evenly (sx8_kv4.h); a piece is a run of blocks of one unit, its four
// waves take every fourth block.  Per block a wave computes S^T = K Q^T on v_mfma_f32_16x16x32_f16 with the tokens as
// rows and the unit's 16 query rows as columns, so that a lane (column c, step group h) holds the scores of
// tokens 4 h + r and 16 + 4 h + r of its own query row and the softmax stays in the lane.  The levels go into the
// MFMA as the fp16 subnormals level * 2^-24, which is one shift and one mask for two values and exact; the scale
// multiplies each group's 32-bit sum (q . k = sum_g s_g (q_g . level_g) + m_g sum(q_g)), and the minima's part is
// one more MFMA with sum(q_g) as two fp16 numbers.  O^T += V^T P^T takes the levels in the same way, with p * s of
// each token rounded to two fp16 numbers (22 bits), and the minima's part sum_t p_t m_t,g as MFMAs of their own.
// So nothing is rounded to fewer than 22 bits between the cache and the output.
// Query rows are multiplied by a power of two that brings their largest value into [64, 128), which is undone in
// the scale: bf16 rows become fp16 without loss (but for values 2^-30 below the largest), and sum(q_g) fits.
// p is kept at or below 8 (the running maximum is raised when a score exceeds it by 3 in powers of two), so p * s
// fits in fp16 for every s.
constexpr int kWgs = 512;                 // two for each of 256 CUs
constexpr float kRaise = 3.f;

struct Kv4Piece {                         // record of a unit cut after this work-group's share: parts == 0: none
    int32_t parts, first_at, tile, head;
    int64_t row0, n;
};
static_assert(sizeof(Kv4Piece) == 32, "record");

struct AttendIo {
    const uint16_t* q;
    uint16_t* out;
    int64_t q_ts, q_hs, o_ts, o_hs;
    float scale_log2;
    float* part_o;                        // [2 kWgs][16][HD]
    float* part_ml;                       // [2 kWgs][16][2]
    Kv4Piece* piece;                      // [kWgs]
};

constexpr int64_t attend_ws(int64_t hd) { return 2 * kWgs * 16 * (hd + 2) * 4 + kWgs * (int64_t)sizeof(Kv4Piece); }

template <int HD>
struct Kv4Regs {                          // a lane's share of one block
    static constexpr int W = HD / 32, NT = HD / 16, NG = HD / kKv4Group;
    uint32_t kw[2][W], vw[NT];
    u32x4 ks[NG], vs[NG], vm;
    uint32_t km[2][(NG + 1) / 2];
    bool bad;
};

__device__ __forceinline__ f16x8 levels(uint32_t w) {
    const u32x4 v = {w & 0x000F000Fu, (w >> 4) & 0x000F000Fu, (w >> 8) & 0x000F000Fu, (w >> 12) & 0x000F000Fu};
    return __builtin_bit_cast(f16x8, v);
}
__device__ __forceinline__ f32x4 mfma16(f16x8 a, f16x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ float max4(float v) {                   // over the lanes of a column
    v = fmaxf(v, __shfl_xor(v, 16, 64));
    return fmaxf(v, __shfl_xor(v, 32, 64));
}
__device__ __forceinline__ float sum4(float v) {
    v += __shfl_xor(v, 16, 64);
    return v + __shfl_xor(v, 32, 64);
}

template <int HD, bool kBf16>
__device__ __forceinline__ void store_row(uint16_t* dst, const float* v) {      // HD / 16 values
    constexpr int N = HD / 16;
    uint32_t w[N / 2];
#pragma unroll
    for (int e = 0; e < N / 2; ++e) w[e] = pack16<kBf16>(v[2 * e], v[2 * e + 1]);
    if constexpr (N == 4) *reinterpret_cast<u32x2*>(dst) = u32x2{w[0], w[1]};
    else
#pragma unroll
        for (int i = 0; i < N / 8; ++i)
            reinterpret_cast<u32x4*>(dst)[i] = u32x4{w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]};
}

template <int HD, bool kBf16>
__global__ __launch_bounds__(256) void k_kv4_attend(const Kv4Pool p, const AttendIo io) {
    using Regs = Kv4Regs<HD>;
    constexpr int W = Regs::W, NT = Regs::NT, NG = Regs::NG, kBB = kv4_block_bytes(HD), kRow = HD + 4;
    constexpr float kInf = __builtin_inff();
    __shared__ __align__(16) float so[4][16][kRow];
    __shared__ float sml[4][16][2];
    int64_t* const pre = reinterpret_cast<int64_t*>(dyn_lds);
    const int tid = threadIdx.x, lane = tid & 63, c = lane & 15, h = lane >> 4;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int S = p.sh.n_slots, G = p.sh.G;
    prefix_sums<256>(S, pre, [&](int s) { return kv4_slot_blocks(p.sh, p.lens, p.cu, s); });
    __syncthreads();
    const int64_t total = uniform(pre[S]), share = kv4_share(total, gridDim.x);
    int64_t x = (int64_t)blockIdx.x * share;
    const int64_t x0 = x, x1 = x + share < total ? x + share : total;
    if (x >= total) {
        if (tid == 0) io.piece[blockIdx.x].parts = 0;
        return;
    }
    int slot = find_item<256>(S, pre, x);
    bool cut = false;
    while (x < x1) {
        while (x >= uniform(pre[slot + 1])) ++slot;
        int64_t row0, n;
        kv4_rows(p.sh, p.cu, slot, &row0, &n);
        row0 = uniform(row0);
        n = uniform(n);
        const int64_t len = uniform(kv4_len(p.sh, p.lens, slot)), nb = kv4_unit_blocks(len), tiles = kv4_tiles(n, G);
        const int64_t off = x - uniform(pre[slot]), unit = off / nb, b0 = off - unit * nb;
        const int64_t bend = nb - b0 < x1 - x ? nb : b0 + (x1 - x);
        const int head = (int)(unit / tiles);
        const int64_t tile = unit - head * tiles;
        // the column's query row, and the last position it may attend
        const int64_t r = 16 * tile + c, tok = r / G;
        const bool row_ok = tok < n;
        const int64_t lim = row_ok ? len - n + tok : len - 1;
        const int64_t tok_min = 16 * tile / G, tok_max = (16 * tile + 15) / G;
        const int64_t lim_min = len - n + tok_min, lim_max = len - n + (tok_max < n ? tok_max : n - 1);
        const int64_t b1 = lim_max < 0 ? b0 : bend < lim_max / 32 + 1 ? bend : lim_max / 32 + 1;   // blocks it reads
        // query fragment: fp16 with the row's largest value in [64, 128)
        f16x8 qf[W], qm;
        float kscale;
        {
            const uint16_t* qr = io.q + (row_ok ? (row0 + tok) * io.q_ts + (head * G + (int)(r - tok * G)) * io.q_hs
                                                : row0 * io.q_ts + head * G * io.q_hs) + 8 * h;
            u32x4 raw[W];
#pragma unroll
            for (int j = 0; j < W; ++j) raw[j] = *reinterpret_cast<const u32x4*>(qr + 32 * j);
            float top = 0.f;
#pragma unroll
            for (int j = 0; j < W; ++j)
#pragma unroll
                for (int e = 0; e < 8; ++e) top = fmaxf(top, __builtin_fabsf(ld16<kBf16>(half_of(raw[j][e >> 1], e))));
            top = max4(row_ok ? top : 0.f);
            // exponent of the largest value; no scaling of rows that are zero or not finite
            const int ex = (int)(__builtin_bit_cast(uint32_t, top) >> 23);
            const int up = top > 0.f && ex < 255 && ex > 0 ? (127 + 6 - ex < 126 ? 127 + 6 - ex : 126) : 0;
            const float mul = __builtin_ldexpf(row_ok ? 1.f : 0.f, up);
            kscale = io.scale_log2 * __builtin_ldexpf(1.f, -up);
            float qs[NG];
#pragma unroll
            for (int g = 0; g < NG; ++g) qs[g] = 0.f;
#pragma unroll
            for (int j = 0; j < W; ++j)
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float raw_q = ld16<kBf16>(half_of(raw[j][e >> 1], e));
                    const _Float16 v = (_Float16)(row_ok ? raw_q * mul : 0.f);
                    qf[j][e] = v;
                    qs[j / 2] += (float)v;
                }
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
        }
        f32x4 o[NT], om = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int t = 0; t < NT; ++t) o[t] = f32x4{0.f, 0.f, 0.f, 0.f};
        float m = -kInf, l = 0.f;
        const int cnt = b1 > b0 + w ? (int)((b1 - b0 - w + 3) / 4) : 0;    // blocks of this wave: b0 + w + 4 i
        int pages = -1;                                                    // lane i: page of block (i0 + i)
        auto load_pages = [&](int i0) {
            const int64_t b = b0 + w + 4 * (int64_t)(i0 + lane);
            pages = b < b1 ? p.table[(int64_t)slot * p.max_pages + (b >> p.bpp_log2)] : -1;
        };
        auto load = [&](Regs& rg, int i) __attribute__((always_inline)) {
            if ((i & 63) == 0) load_pages(i);
            const int64_t b = b0 + w + 4 * (int64_t)i;
            int page = __builtin_amdgcn_readlane(pages, i & 63);
            rg.bad = page < 0 || page >= p.n_pages;
            page = rg.bad ? 0 : page;
            const uint8_t* base = p.pages + page * p.page_bytes
                + (((int64_t)head << p.bpp_log2) + (b & ((1 << p.bpp_log2) - 1))) * kBB;
            const uint8_t* prm = base + 32 * HD;
            if constexpr (W == 2) {
#pragma unroll
                for (int a = 0; a < 2; ++a) {
                    const u32x2 v = *reinterpret_cast<const u32x2*>(base + a * 512 + lane * 8);
                    rg.kw[a][0] = v.x;
                    rg.kw[a][1] = v.y;
                }
            } else {
#pragma unroll
                for (int a = 0; a < 2; ++a)
#pragma unroll
                    for (int q4 = 0; q4 < W / 4; ++q4) {
                        const u32x4 v = *reinterpret_cast<const u32x4*>(base + a * (256 * W) + q4 * 1024 + lane * 16);
#pragma unroll
                        for (int e = 0; e < 4; ++e) rg.kw[a][4 * q4 + e] = v[e];
                    }
            }
#pragma unroll
            for (int g = 0; g < NG; ++g) rg.ks[g] = *reinterpret_cast<const u32x4*>(prm + (g * 32 + h * 8) * 2);
#pragma unroll
            for (int a = 0; a < 2; ++a) {
                const uint8_t* at = prm + NG * 64 + (16 * a + c) * NG * 2;
                if constexpr (NG == 1) rg.km[a][0] = *reinterpret_cast<const uint16_t*>(at);
                else if constexpr (NG == 2) rg.km[a][0] = *reinterpret_cast<const uint32_t*>(at);
                else {
                    const u32x2 v = *reinterpret_cast<const u32x2*>(at);
                    rg.km[a][0] = v.x;
                    rg.km[a][1] = v.y;
                }
            }
#pragma unroll
            for (int q4 = 0; q4 < NT / 4; ++q4) {
                const u32x4 v = *reinterpret_cast<const u32x4*>(base + 16 * HD + q4 * 1024 + lane * 16);
#pragma unroll
                for (int e = 0; e < 4; ++e) rg.vw[4 * q4 + e] = v[e];
            }
#pragma unroll
            for (int g = 0; g < NG; ++g)
                rg.vs[g] = *reinterpret_cast<const u32x4*>(prm + 2 * NG * 64 + (g * 32 + h * 8) * 2);
            rg.vm = *reinterpret_cast<const u32x4*>(prm + 3 * NG * 64 + ((c < NG ? c : 0) * 32 + h * 8) * 2);
        };
        // kMask: the block reaches past a column's last position, or has no page
        auto block = [&](Regs& rg, int64_t b, auto mask) __attribute__((always_inline)) {
            constexpr bool kMask = decltype(mask)::value;
            float sc[8];
#pragma unroll
            for (int a = 0; a < 2; ++a) {
                f32x4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int g = 0; g < NG; ++g) {
                    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
                    acc = mfma16(levels(rg.kw[a][2 * g]), qf[2 * g], acc);
                    acc = mfma16(levels(rg.kw[a][2 * g + 1]), qf[2 * g + 1], acc);
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        s[e] = __builtin_fmaf(sx8_h2f(half_of(rg.ks[g][2 * a + (e >> 1)], e)), acc[e], s[e]);
                }
                u32x4 mw = {0u, 0u, 0u, 0u};
                if (h == 0) {
                    mw.x = rg.km[a][0];
                    mw.z = rg.km[a][0];
                    if constexpr (NG == 4) mw.y = mw.w = rg.km[a][1];
                }
                const f32x4 mt = mfma16(__builtin_bit_cast(f16x8, mw), qm, f32x4{0.f, 0.f, 0.f, 0.f});
#pragma unroll
                for (int e = 0; e < 4; ++e) sc[4 * a + e] = __builtin_fmaf(s[e], 16777216.f, mt[e]);
            }
            if constexpr (kMask) {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const int64_t key = b * 32 + (e / 4) * 16 + 4 * h + e % 4;
                    sc[e] = key <= lim && !rg.bad ? sc[e] : -kInf;
                }
            }
            float mx = sc[0];
#pragma unroll
            for (int e = 1; e < 8; ++e) mx = fmaxf(mx, sc[e]);
            mx *= kscale;
            if (__builtin_amdgcn_ballot_w64(mx > m + kRaise) != 0) {
                const float mn = fmaxf(m, max4(mx));
                const float alpha = m == mn ? 1.f : __builtin_amdgcn_exp2f(m - mn);
                m = mn;
                l *= alpha;
                om *= alpha;
#pragma unroll
                for (int t = 0; t < NT; ++t) o[t] *= alpha;
            }
            const float nm = m == -kInf ? 0.f : -m;
            float pv[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                pv[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[e], kscale, nm));
                l += pv[e];
            }
            u32x4 vm = rg.vm;
            if (c >= NG) vm = u32x4{0u, 0u, 0u, 0u};
            if constexpr (kMask) {
                // a token that some column may not attend must not reach it through 0 * NaN: its minimum is zero where
                // it is no number (the scale, which is none either, still brings the NaN to the columns that attend it)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const uint32_t lo = vm[e] & 0x7FFFu, hi = vm[e] >> 16 & 0x7FFFu;
                    vm[e] = (lo >= 0x7C00u ? 0u : vm[e] & 0xFFFFu) | (hi >= 0x7C00u ? 0u : vm[e] & 0xFFFF0000u);
                }
            }
            f16x8 ph, pl;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                ph[e] = (_Float16)pv[e];
                pl[e] = (_Float16)(pv[e] - (float)ph[e]);
            }
            const f16x8 vm8 = __builtin_bit_cast(f16x8, vm);
            om = mfma16(vm8, ph, om);
            om = mfma16(vm8, pl, om);
#pragma unroll
            for (int g = 0; g < NG; ++g) {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float s = sx8_h2f(half_of(rg.vs[g][e >> 1], e));
                    const float ps = kMask && pv[e] == 0.f ? 0.f : s;
                    ph[e] = (_Float16)(pv[e] * ps);
                    pl[e] = (_Float16)__builtin_fmaf(pv[e], ps, -(float)ph[e]);
                }
#pragma unroll
                for (int t = 4 * g; t < 4 * g + 4; ++t) {
                    const f16x8 lv = levels(rg.vw[t]);
                    o[t] = mfma16(lv, ph, o[t]);
                    o[t] = mfma16(lv, pl, o[t]);
                }
            }
        };
        auto step = [&](Regs& rg, int i) __attribute__((always_inline)) {
            const int64_t b = b0 + w + 4 * (int64_t)i;
            if (b * 32 + 31 > lim_min || rg.bad) block(rg, b, std::true_type{});
            else block(rg, b, std::false_type{});
        };
        Regs r0, r1;
        if (cnt > 0) load(r0, 0);
        for (int i = 0; i < cnt; i += 2) {
            if (i + 1 < cnt) load(r1, i + 1);
            step(r0, i);
            if (i + 1 >= cnt) break;
            if (i + 2 < cnt) load(r0, i + 2);
            step(r1, i + 1);
        }
        // the four waves' states meet in LDS: O = 2^24 (levels) + (minima's sum of the group, row g of om)
        l = sum4(l);
        float og[NG];
#pragma unroll
        for (int g = 0; g < NG; ++g) og[g] = __shfl(om[g], c, 64);
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            f32x4 v;
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = __builtin_fmaf(o[t][e], 16777216.f, og[t / 4]);
            *reinterpret_cast<f32x4*>(&so[w][c][16 * t + 4 * h]) = v;
        }
        if (h == 0) {
            sml[w][c][0] = m;
            sml[w][c][1] = l;
        }
        __syncthreads();
        {
            constexpr int N = HD / 16;
            const int col = tid >> 4, d0 = (tid & 15) * N;
            float mm = sml[0][col][0];
#pragma unroll
            for (int i = 1; i < 4; ++i) mm = fmaxf(mm, sml[i][col][0]);
            float den = 0.f, acc[N];
#pragma unroll
            for (int e = 0; e < N; ++e) acc[e] = 0.f;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float f = sml[i][col][0] == mm ? 1.f : __builtin_amdgcn_exp2f(sml[i][col][0] - mm);
                den = __builtin_fmaf(f, sml[i][col][1], den);
#pragma unroll
                for (int e = 0; e < N; ++e) acc[e] = __builtin_fmaf(f, so[i][col][d0 + e], acc[e]);
            }
            const int64_t rr = 16 * tile + col, tk = rr / G;
            if (b0 == 0 && bend == nb) {
                if (tk < n) {
                    const float inv = den == 0.f ? 0.f : 1.f / den;
#pragma unroll
                    for (int e = 0; e < N; ++e) acc[e] *= inv;
                    store_row<HD, kBf16>(io.out + (row0 + tk) * io.o_ts + (head * G + (int)(rr - tk * G)) * io.o_hs + d0,
                                         acc);
                }
            } else {
                const int64_t at = 2 * (int64_t)blockIdx.x + (x == x0 ? 0 : 1);
                float* po = io.part_o + (at * 16 + col) * HD + d0;
#pragma unroll
                for (int e = 0; e < N; e += 4)
                    *reinterpret_cast<f32x4*>(po + e) = f32x4{acc[e], acc[e + 1], acc[e + 2], acc[e + 3]};
                if ((tid & 15) == 0) {
                    io.part_ml[(at * 16 + col) * 2] = mm;
                    io.part_ml[(at * 16 + col) * 2 + 1] = den;
                }
            }
        }
        // a unit whose first piece this is and that goes on in the next work-groups: its record for the combine
        if (bend < nb && x - b0 >= x0) {
            cut = true;
            if (tid == 0) {
                Kv4Piece pc;
                pc.parts = (int32_t)((x - b0 + nb - 1) / share - blockIdx.x + 1);
                pc.first_at = x == x0 ? 0 : 1;
                pc.tile = (int32_t)tile;
                pc.head = head;
                pc.row0 = row0;
                pc.n = n;
                io.piece[blockIdx.x] = pc;
            }
        }
        x += bend - b0;
        __syncthreads();
    }
    if (!cut && tid == 0) io.piece[blockIdx.x].parts = 0;
}

// Units that were cut: work-group i merges the unit whose first piece ends the share of work-group i, its parts in their
// order (part 0 at slot 2 i + first_at, the next ones at 2 (i + 1), 2 (i + 2), ...).  Wave = (row, quarter of the parts).
template <int HD, bool kBf16>
__global__ __launch_bounds__(1024) void k_kv4_combine(const AttendIo io, int G) {
    constexpr int N = HD / 64;
    const Kv4Piece pc = io.piece[blockIdx.x];
    if (pc.parts == 0) return;
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), quarter = w & 3;
    const int row = 4 * blockIdx.y + (w >> 2);
    const int64_t rr = 16 * (int64_t)pc.tile + row, tk = rr / G;
    const bool live = tk < pc.n;
    __shared__ float sml[16][2], so[16][HD];
    auto at = [&](int i) { return (2 * ((int64_t)blockIdx.x + i) + (i == 0 ? pc.first_at : 0)) * 16 + row; };
    const int per = (pc.parts + 3) / 4, i0 = quarter * per, i1 = min(i0 + per, pc.parts);
    float m = -__builtin_inff();
    if (live) {
        for (int i = i0 + lane; i < i1; i += 64) m = fmaxf(m, io.part_ml[at(i) * 2]);
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
    }
    float den = 0.f, acc[N];
#pragma unroll
    for (int e = 0; e < N; ++e) acc[e] = 0.f;
    if (live) {
        constexpr int kU = 8;                       // parts requested together
        for (int i = i0; i < i1; i += kU) {
            float v[kU][N], pm[kU], pl[kU];
#pragma unroll
            for (int u = 0; u < kU; ++u) {
                const int64_t a = at(min(i + u, i1 - 1));
                pm[u] = io.part_ml[a * 2];
                pl[u] = io.part_ml[a * 2 + 1];
#pragma unroll
                for (int e = 0; e < N; ++e) v[u][e] = io.part_o[a * HD + 64 * e + lane];
            }
#pragma unroll
            for (int u = 0; u < kU; ++u) {
                if (i + u >= i1) break;
                const float f = pm[u] == m ? 1.f : __builtin_amdgcn_exp2f(pm[u] - m);
                den = __builtin_fmaf(f, pl[u], den);
#pragma unroll
                for (int e = 0; e < N; ++e) acc[e] = __builtin_fmaf(f, v[u][e], acc[e]);
            }
        }
    }
    if (lane == 0) {
        sml[w][0] = m;
        sml[w][1] = den;
    }
#pragma unroll
    for (int e = 0; e < N; ++e) so[w][64 * e + lane] = acc[e];
    __syncthreads();
    if (quarter != 0 || !live) return;
    float mm = m;
#pragma unroll
    for (int i = 1; i < 4; ++i) mm = fmaxf(mm, sml[w + i][0]);
    const float f0 = m == mm ? 1.f : __builtin_amdgcn_exp2f(m - mm);
    den *= f0;
#pragma unroll
    for (int e = 0; e < N; ++e) acc[e] *= f0;
#pragma unroll
    for (int i = 1; i < 4; ++i) {
        const float f = sml[w + i][0] == mm ? 1.f : __builtin_amdgcn_exp2f(sml[w + i][0] - mm);
        den = __builtin_fmaf(f, sml[w + i][1], den);
#pragma unroll
        for (int e = 0; e < N; ++e) acc[e] = __builtin_fmaf(f, so[w + i][64 * e + lane], acc[e]);
    }
    const float inv = den == 0.f ? 0.f : 1.f / den;
    uint16_t* dst = io.out + (pc.row0 + tk) * io.o_ts + (pc.head * G + (int)(rr - tk * G)) * io.o_hs;
#pragma unroll
    for (int e = 0; e < N; ++e) dst[64 * e + lane] = (uint16_t)st16<kBf16>(acc[e] * inv);
}

// ---- host --------------------------------------------------------------------------------------
bool hd_ok(int hd) { return hd == 64 || hd == 128 || hd == 256; }

int32_t make_pool(const char* what, Kv4Pool* p, const uint8_t* pages, const int32_t* table, const int32_t* lens,
                  const int32_t* cu, int64_t n_slots, int64_t max_pages, int64_t n_pages, int64_t rows, int32_t nk,
                  int32_t hd, int32_t page_tokens, int32_t dtype) {
    if (!pages || !table || !lens) return fail(SX8_ERR_INVALID, "%s: null pointer", what);
    const int64_t pb = sx8_kv4_page_bytes(nk, hd, page_tokens);
    if (pb < 0)
        return fail(SX8_ERR_INVALID, "%s: bad shape (hd 64, 128 or 256, page_tokens 32, 64, 128 or 256, 1 <= nk <= 256)",
                    what);
    if (n_slots <= 0 || n_slots > kKv4MaxSlots || max_pages <= 0 || max_pages * page_tokens > kKv4MaxTokens ||
        n_pages <= 0 || n_pages > 0x7FFFFFFF)
        return fail(SX8_ERR_INVALID, "%s: bad sizes (n_slots 1..%d, max_pages * page_tokens 1..%lld, n_pages)", what,
                    kKv4MaxSlots, (long long)kKv4MaxTokens);
    if (rows < 0 || rows > 0x7FFFFFFF || (!cu && rows != n_slots))
        return fail(SX8_ERR_INVALID, "%s: bad rows (without cu one row a slot)", what);
    if (!aligned(pages, 16) || !aligned(table, 4) || !aligned(lens, 4) || !aligned(cu, 4))
        return fail(SX8_ERR_INVALID, "%s: pages must be 16-byte aligned, table, lens and cu 4-byte", what);
    if (dtype != 0 && dtype != 1) return fail(SX8_ERR_INVALID, "%s: dtype must be 0 (fp16) or 1 (bf16)", what);
    p->pages = pages;
    p->table = table;
    p->lens = lens;
    p->cu = cu;
    p->page_bytes = pb;
    p->max_pages = (int)max_pages;
    p->n_pages = (int)n_pages;
    p->bpp_log2 = page_tokens == 32 ? 0 : page_tokens == 64 ? 1 : page_tokens == 128 ? 2 : 3;
    p->sh = Kv4Shape{(int)n_slots, nk, 1, max_pages * page_tokens, rows};
    return SX8_OK;
}

// Row pointers (null: only without rows): 16-byte aligned, strides multiples of 8.
int32_t check_rows(const char* what, const char* name, const void* ptr, int64_t ts, int64_t hs, int64_t rows) {
    if (!ptr && rows > 0) return fail(SX8_ERR_INVALID, "%s: null pointer", what);
    if (!aligned(ptr, 16) || ts % 8 || hs % 8 || ts < 0 || hs < 0 || ts > (int64_t)1 << 40 || hs > (int64_t)1 << 40)
        return fail(SX8_ERR_INVALID, "%s: %s must be 16-byte aligned with strides that are multiples of 8", what, name);
    return SX8_OK;
}

// f(integral_constant<hd>, integral_constant<bf16>)
template <typename F>
void by_kind(int hd, int dtype, F&& f) {
    auto with = [&](auto d) {
        if (dtype) f(d, std::true_type{});
        else f(d, std::false_type{});
    };
    if (hd == 64) with(std::integral_constant<int, 64>{});
    else if (hd == 128) with(std::integral_constant<int, 128>{});
    else with(std::integral_constant<int, 256>{});
}

unsigned prefix_bytes(const Kv4Pool& p) { return (unsigned)(p.sh.n_slots + 1) * 8; }

}  // namespace
}  // namespace sx8

extern "C" int64_t sx8_kv4_page_bytes(int32_t nk, int32_t hd, int32_t page_tokens) {
    using namespace sx8;
    if (nk < 1 || nk > 256 || !hd_ok(hd) || (page_tokens != 32 && page_tokens != 64 && page_tokens != 128 && page_tokens != 256))
        return -1;
    return (int64_t)nk * (page_tokens / 32) * kv4_block_bytes(hd);
}

extern "C" int32_t sx8_kv4_append(uint8_t* pages, const int32_t* table, const int32_t* lens, const int32_t* cu,
                                  int64_t n_slots, int64_t max_pages, int64_t n_pages, const void* k, const void* v,
                                  int64_t rows, int64_t k_ts, int64_t k_hs, int64_t v_ts, int64_t v_hs, int32_t nk,
                                  int32_t hd, int32_t page_tokens, int32_t dtype, void* stream) {
    using namespace sx8;
    const char* what = "sx8_kv4_append";
    Kv4Pool p;
    int32_t rc = make_pool(what, &p, pages, table, lens, cu, n_slots, max_pages, n_pages, rows, nk, hd, page_tokens, dtype);
    if (rc == SX8_OK) rc = check_rows(what, "k", k, k_ts, k_hs, rows);
    if (rc == SX8_OK) rc = check_rows(what, "v", v, v_ts, v_hs, rows);
    if (rc != SX8_OK) return rc;
    if (rows == 0) return ok();
    const RowsIn in{(const uint16_t*)k, (const uint16_t*)v, k_ts, k_hs, v_ts, v_hs};
    const dim3 grid((unsigned)kv4_touched_most(n_slots, rows, cu != nullptr), (unsigned)nk);
    by_kind(hd, dtype, [&](auto d, auto b) {
        hipLaunchKernelGGL((k_kv4_append<decltype(d)::value, decltype(b)::value>), grid, dim3(256), prefix_bytes(p),
                           as_stream(stream), p, in);
    });
    return check_launch(what);
}

extern "C" int32_t sx8_kv4_read(const uint8_t* pages, const int32_t* table, const int32_t* lens, const int32_t* cu,
                                int64_t n_slots, int64_t max_pages, int64_t n_pages, void* k, void* v, int64_t rows,
                                int64_t k_ts, int64_t k_hs, int64_t v_ts, int64_t v_hs, int32_t nk, int32_t hd,
                                int32_t page_tokens, int32_t dtype, void* stream) {
    using namespace sx8;
    const char* what = "sx8_kv4_read";
    Kv4Pool p;
    int32_t rc = make_pool(what, &p, pages, table, lens, cu, n_slots, max_pages, n_pages, rows, nk, hd, page_tokens, dtype);
    if (rc == SX8_OK) rc = check_rows(what, "k", k, k_ts, k_hs, rows);
    if (rc == SX8_OK) rc = check_rows(what, "v", v, v_ts, v_hs, rows);
    if (rc != SX8_OK) return rc;
    if (rows == 0) return ok();
    const RowsOut out{(uint16_t*)k, (uint16_t*)v, k_ts, k_hs, v_ts, v_hs};
    const dim3 grid((unsigned)kv4_touched_most(n_slots, rows, cu != nullptr), (unsigned)nk);
    by_kind(hd, dtype, [&](auto d, auto b) {
        hipLaunchKernelGGL((k_kv4_read<decltype(d)::value, decltype(b)::value>), grid, dim3(256), prefix_bytes(p),
                           as_stream(stream), p, out);
    });
    return check_launch(what);
}

extern "C" int64_t sx8_kv4_attend_workspace_bytes(int32_t hd) { return sx8::hd_ok(hd) ? sx8::attend_ws(hd) : -1; }

extern "C" int32_t sx8_kv4_attend(const uint8_t* pages, const int32_t* table, const int32_t* lens, const int32_t* cu,
                                  int64_t n_slots, int64_t max_pages, int64_t n_pages, const void* q, void* out,
                                  int64_t rows, int64_t q_ts, int64_t q_hs, int64_t o_ts, int64_t o_hs, int32_t nh,
                                  int32_t nk, int32_t hd, int32_t page_tokens, float scale, int32_t dtype,
                                  void* workspace, int64_t workspace_bytes, void* stream) {
    using namespace sx8;
    const char* what = "sx8_kv4_attend";
    Kv4Pool p;
    int32_t rc = make_pool(what, &p, pages, table, lens, cu, n_slots, max_pages, n_pages, rows, nk, hd, page_tokens, dtype);
    if (rc == SX8_OK) rc = check_rows(what, "q", q, q_ts, q_hs, rows);
    if (rc == SX8_OK) rc = check_rows(what, "out", out, o_ts, o_hs, rows);
    if (rc != SX8_OK) return rc;
    if (nh <= 0 || nh % nk || nh / nk > 256)
        return fail(SX8_ERR_INVALID, "%s: nh must be a multiple of nk, at most 256 nk", what);
    if (!(scale > 0.f) || !(scale < __builtin_inff()))
        return fail(SX8_ERR_INVALID, "%s: scale must be positive and finite", what);
    if (!workspace || workspace_bytes < attend_ws(hd) || !aligned(workspace, 256))
        return fail(SX8_ERR_INVALID, "%s: workspace needs %lld bytes, 256-byte aligned", what, (long long)attend_ws(hd));
    if (rows == 0) return ok();
    p.sh.G = nh / nk;
    AttendIo io{(const uint16_t*)q, (uint16_t*)out, q_ts, q_hs, o_ts, o_hs, scale * 1.4426950408889634f, nullptr, nullptr,
                nullptr};
    io.piece = reinterpret_cast<Kv4Piece*>(workspace);
    io.part_o = reinterpret_cast<float*>(io.piece + kWgs);
    io.part_ml = io.part_o + 2 * kWgs * 16 * (int64_t)hd;
    // rows of a unit that can be in use: all 16, or those of one token a slot
    const int64_t used = cu ? rows * p.sh.G : p.sh.G;
    const unsigned groups = (unsigned)((used < 16 ? used : 16) + 3) / 4;
    by_kind(hd, dtype, [&](auto d, auto b) {
        hipLaunchKernelGGL((k_kv4_attend<decltype(d)::value, decltype(b)::value>), dim3(kWgs), dim3(256), prefix_bytes(p),
                           as_stream(stream), p, io);
        hipLaunchKernelGGL((k_kv4_combine<decltype(d)::value, decltype(b)::value>), dim3(kWgs, groups), dim3(1024), 0,
                           as_stream(stream), io, p.sh.G);
    });
    return check_launch(what);
}
