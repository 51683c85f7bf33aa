// sx8_kv4_core.h -- what the kernels over the paged 4-bit cache share: the slots' blocks, the encoder of a group, a block's
// registers and their matrix products, and the host's checks (sx8_kv4.hip, sx8_kv4_rope.hip, sx8_kv4_tree.hip).
#pragma once
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
__device__ __forceinline__ int64_t block_offset(const Kv4Pool& p, int slot, int head, int b, int bb) {
    const int at = b >> p.bpp_log2;
    if (b < 0 || at >= p.max_pages) return -1;
    const int page = p.table[(int64_t)slot * p.max_pages + at];
    if (page < 0 || page >= p.n_pages) return -1;
    return page * p.page_bytes + (((int64_t)head << p.bpp_log2) + (b & ((1 << p.bpp_log2) - 1))) * bb;
}

// ---- encoding ----------------------------------------------------------------------------------
struct Enc {
    float s, m;
    uint32_t lv[8];               // kLevel0 + level
};
constexpr uint32_t kLevel0 = 0x4B400000u;      // 1.5 2^23 as a float: adding it rounds to an integer, in the low bits

// The level of x: (x - m) / s to the nearest, ties to even, in exact arithmetic.  The quotient in binary64 is at most one
// level off (bf16's x - m is rounded where x is far smaller than m), and x lies on one side or the other of the borders of its
// level, m + (q +- 1/2) s, which are exact: multiples of 2^-25 below 2^21.
__device__ __noinline__ uint32_t exact_level(float x, float m, float s) {
#pragma clang fp contract(off)
    const double v = x, m64 = m, s64 = s;
    double q = __builtin_rint((v - m64) / s64);
    const double above = m64 + (q + 0.5) * s64, below = m64 + (q - 0.5) * s64;
    const bool odd = (int)q & 1;
    if (v > above || (v == above && odd)) q += 1.0;
    else if (v < below || (v == below && odd)) q -= 1.0;
    return kLevel0 + (uint32_t)(int)fmin(fmax(q, 0.0), 15.0);
}

// x[i] - m of the eight rows' values (fp16: without a conversion of its own)
template <bool kBf16, int kHalf>
__device__ __forceinline__ float less(uint32_t word, float m) {
    if constexpr (kBf16) return ld16<true>(half_of(word, kHalf)) - m;
    float d;
    if constexpr (kHalf) asm("v_fma_mix_f32 %0, %1, 1.0, -%2 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(d) : "v"(word), "v"(m));
    else asm("v_fma_mix_f32 %0, %1, 1.0, -%2 op_sel:[0,0,0] op_sel_hi:[1,0,0]" : "=v"(d) : "v"(word), "v"(m));
    return d;
}

// The ends of a group come from integers that order as the values do (infinities and NaN beyond all others), the minimum and
// the complement of the maximum in one word.  In binary32 the quotient is within 2^-17 of the true one (a fifteenth of it is
// within 2.5 2^-23 of itself: three roundings, and a reciprocal good to one place), so only a quotient within 2^-16 of a
// border is decided by exact_level: one look for the lane's eight values.  (A look for each of them, and the ends in
// binary32: 13081 rows of 8 heads of 128, K and V, 27 us; all quotients in binary64: 50.)
// Rows outside the call come as zeros (their results are unused).
template <bool kBf16>
__device__ __forceinline__ void encode_group(const u32x4& raw, Enc& e) {
#pragma clang fp contract(off)
    typedef int16_t i16x2 __attribute__((ext_vector_type(2)));
    constexpr int kLowest = ~(kBf16 ? 0x7F80 : 0x7C00);          // -infinity
    auto ordered = [](uint32_t w) {
        const uint32_t sign = __builtin_bit_cast(uint32_t, (i16x2)(__builtin_bit_cast(i16x2, w) >> 15));
        return w ^ (sign & 0x7FFF7FFFu);
    };
    auto least = [](uint32_t a, uint32_t b) {
        return __builtin_bit_cast(uint32_t, __builtin_elementwise_min(__builtin_bit_cast(i16x2, a), __builtin_bit_cast(i16x2, b)));
    };
    uint32_t lows = ordered(raw[0]), highs = ~lows;
#pragma unroll
    for (int i = 1; i < 4; ++i) {
        const uint32_t w = ordered(raw[i]);
        lows = least(lows, w);
        highs = least(highs, ~w);
    }
    // low half: the minimum, high half: the complement of the maximum; over the eight lanes of the group
    uint32_t ends = least(__builtin_amdgcn_perm(highs, lows, 0x05040100u), __builtin_amdgcn_perm(highs, lows, 0x07060302u));
    ends = least(ends, __builtin_amdgcn_mov_dpp((int)ends, 0xB1, 0xF, 0xF, true));
    ends = least(ends, __builtin_amdgcn_mov_dpp((int)ends, 0x4E, 0xF, 0xF, true));
    ends = least(ends, __builtin_amdgcn_mov_dpp((int)ends, 0x141, 0xF, 0xF, true));
    const bool none = min((int)(int16_t)ends, (int)ends >> 16) <= kLowest;
    const uint32_t both = ordered(ends ^ 0xFFFF0000u);
    const float lo = ld16<kBf16>(both & 0xFFFFu), r = ld16<kBf16>(both >> 16) - lo;
    e.s = none ? __builtin_nanf("") : (float)(_Float16)fminf(r * (1.0f / 15.0f), 65504.0f);
    e.m = none ? __builtin_nanf("") : (float)(_Float16)fminf(fmaxf(lo, -65504.0f), 65504.0f);
    const float part = e.s > 0.f ? __builtin_amdgcn_rcpf(e.s) * (1.0f / 15.0f) : 0.f;
    const float big = __builtin_bit_cast(float, kLevel0);
    float off[8], far = 0.f;
    auto level = [&](int i, float d) {
        const float u = fminf(fmaxf(d * part, 0.f), 1.f);        // (NaN: 0)
        const float n = __builtin_fmaf(u, 15.f, big);
        e.lv[i] = __builtin_bit_cast(uint32_t, n);
        off[i] = __builtin_fmaf(u, 15.f, big - n);
        far = fmaxf(far, __builtin_fabsf(off[i]));
    };
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        level(2 * i, less<kBf16, 0>(raw[i], e.m));
        level(2 * i + 1, less<kBf16, 1>(raw[i], e.m));
    }
    if (far >= 0.5f - 0x1p-16f) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (__builtin_fabsf(off[i]) >= 0.5f - 0x1p-16f) e.lv[i] = exact_level(ld16<kBf16>(half_of(raw[i >> 1], i)), e.m, e.s);
    }
}

// The block that work item `item` of the call names: slot, its block, and the new tokens in it (block-relative
// [t0, t1), row of token t0).  Every wave finds it; false past the last item.
struct Touched {
    int slot, block, t0, t1, row0;
    int first;                              // the slot's tokens before its new ones (below zero: more rows than tokens)
};
__device__ __forceinline__ bool find_touched(const Kv4Pool& p, int64_t item, int64_t* pre, Touched* t) {
    const int S = p.sh.n_slots, lane = threadIdx.x & 63;
    int first, n, len, b;
    int64_t before;
    auto count = [&](int s) {
        kv4_rows(p.sh, p.cu, s, &first, &n);
        len = kv4_len(p.sh, p.lens, s);
        return (int64_t)kv4_touched(len, n, &b);
    };
    if (!p.cu) {                            // one row a slot touches one block
        t->slot = (int)item;
        before = item;
        count(t->slot);
    } else if (S <= 64) {
        const int64_t mine = lane < S ? count(lane) : 0, end = wave_prefix(mine);
        const uint64_t past = __builtin_amdgcn_ballot_w64(lane < S && end <= item);
        t->slot = __builtin_popcountll(past);
        if (t->slot >= S) return false;
        before = lane_of(end - mine, t->slot);
        first = __builtin_amdgcn_readlane(first, t->slot);
        n = __builtin_amdgcn_readlane(n, t->slot);
        len = __builtin_amdgcn_readlane(len, t->slot);
    } else {
        prefix_sums<256>(S, pre, count);
        __syncthreads();
        if (item >= uniform(pre[S])) return false;
        t->slot = find_item<256>(S, pre, item);
        before = uniform(pre[t->slot]);
        count(t->slot);
    }
    first = __builtin_amdgcn_readfirstlane(first);
    n = __builtin_amdgcn_readfirstlane(n);
    len = __builtin_amdgcn_readfirstlane(len);
    kv4_touched(len, n, &b);
    t->block = b + (int)(item - before);
    const int a = max(len - n, t->block * 32), e = min(len, t->block * 32 + 32);
    t->t0 = a - t->block * 32;
    t->t1 = e - t->block * 32;
    t->row0 = first + a - (len - n);
    t->first = len - n;
    return true;
}

struct RowsIn {
    const uint16_t* k;
    const uint16_t* v;
    int64_t k_ts, k_hs, v_ts, v_hs;
};

extern __shared__ __align__(16) unsigned char dyn_lds[];

// ---- attention ---------------------------------------------------------------------------------
// How far the running maximum lies below the largest score, and how far a score may exceed it (sx8_kv4.hip: why).
constexpr float kUp = 10.f, kSlack = 3.f;

template <int HD>
struct Kv4Regs {                          // a lane's share of one block
    static constexpr int W = HD / 32, NT = HD / 16, NG = HD / kKv4Group;
    uint32_t kw[2][W], vw[NT];
    u32x4 ks[NG], vs[NG], vm;
    uint32_t km[2][(NG + 1) / 2];
    bool bad;
};
// A lane's share of the block at `base`: K's words and parameters, and V's.
template <int HD>
__device__ __forceinline__ void load_block_k(Kv4Regs<HD>& rg, const uint8_t* base, int lane) {
    constexpr int W = Kv4Regs<HD>::W, NG = Kv4Regs<HD>::NG;
    const int c = lane & 15, h = lane >> 4;
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
}
template <int HD>
__device__ __forceinline__ void load_block_v(Kv4Regs<HD>& rg, const uint8_t* base, int lane) {
    constexpr int NT = Kv4Regs<HD>::NT, NG = Kv4Regs<HD>::NG;
    const int c = lane & 15, h = lane >> 4;
    const uint8_t* prm = base + 32 * HD;
#pragma unroll
    for (int q4 = 0; q4 < NT / 4; ++q4) {
        const u32x4 v = *reinterpret_cast<const u32x4*>(base + 16 * HD + q4 * 1024 + lane * 16);
#pragma unroll
        for (int e = 0; e < 4; ++e) rg.vw[4 * q4 + e] = v[e];
    }
#pragma unroll
    for (int g = 0; g < NG; ++g) rg.vs[g] = *reinterpret_cast<const u32x4*>(prm + 2 * NG * 64 + (g * 32 + h * 8) * 2);
    rg.vm = *reinterpret_cast<const u32x4*>(prm + 3 * NG * 64 + ((c < NG ? c : 0) * 32 + h * 8) * 2);
}
template <int HD>
__device__ __forceinline__ void load_block(Kv4Regs<HD>& rg, const uint8_t* base, int lane) {
    load_block_k<HD>(rg, base, lane);
    load_block_v<HD>(rg, base, lane);
}

__device__ __forceinline__ f16x8 levels(uint32_t w) {
    const u32x4 v = {w << 4 & 0x00F000F0u, w & 0x00F000F0u, w >> 4 & 0x00F000F0u, w >> 8 & 0x00F000F0u};
    return __builtin_bit_cast(f16x8, v);
}
// p s of eight values (s: four words of fp16) as two fp16 numbers each, hi + lo: an instruction for each number, where the
// compiler takes three.  The compiler does not see what an asm block reads and writes at its ends, so the waits are here: one
// state between an exp2 and its use, two between the last word and an MFMA that reads it.  (A word's halves, and a number and
// its use, are written four instructions apart from each other.)
__device__ __forceinline__ void split8(const float* p, const u32x4& s, u32x4* hi, u32x4* lo) {
    uint32_t a[4], b[4];
    asm("s_nop 0\n\t"
        "v_fma_mixlo_f16 %0, %8, %16, 0 op_sel:[0,0,0] op_sel_hi:[0,1,0]\n\t"
        "v_fma_mixlo_f16 %1, %10, %17, 0 op_sel:[0,0,0] op_sel_hi:[0,1,0]\n\t"
        "v_fma_mixlo_f16 %2, %12, %18, 0 op_sel:[0,0,0] op_sel_hi:[0,1,0]\n\t"
        "v_fma_mixlo_f16 %3, %14, %19, 0 op_sel:[0,0,0] op_sel_hi:[0,1,0]\n\t"
        "v_fma_mixhi_f16 %0, %9, %16, 0 op_sel:[0,1,0] op_sel_hi:[0,1,0]\n\t"
        "v_fma_mixhi_f16 %1, %11, %17, 0 op_sel:[0,1,0] op_sel_hi:[0,1,0]\n\t"
        "v_fma_mixhi_f16 %2, %13, %18, 0 op_sel:[0,1,0] op_sel_hi:[0,1,0]\n\t"
        "v_fma_mixhi_f16 %3, %15, %19, 0 op_sel:[0,1,0] op_sel_hi:[0,1,0]\n\t"
        "v_fma_mixlo_f16 %4, %8, %16, -%0 op_sel:[0,0,0] op_sel_hi:[0,1,1]\n\t"
        "v_fma_mixlo_f16 %5, %10, %17, -%1 op_sel:[0,0,0] op_sel_hi:[0,1,1]\n\t"
        "v_fma_mixlo_f16 %6, %12, %18, -%2 op_sel:[0,0,0] op_sel_hi:[0,1,1]\n\t"
        "v_fma_mixlo_f16 %7, %14, %19, -%3 op_sel:[0,0,0] op_sel_hi:[0,1,1]\n\t"
        "v_fma_mixhi_f16 %4, %9, %16, -%0 op_sel:[0,1,1] op_sel_hi:[0,1,1]\n\t"
        "v_fma_mixhi_f16 %5, %11, %17, -%1 op_sel:[0,1,1] op_sel_hi:[0,1,1]\n\t"
        "v_fma_mixhi_f16 %6, %13, %18, -%2 op_sel:[0,1,1] op_sel_hi:[0,1,1]\n\t"
        "v_fma_mixhi_f16 %7, %15, %19, -%3 op_sel:[0,1,1] op_sel_hi:[0,1,1]\n\t"
        "s_nop 1"
        : "=&v"(a[0]), "=&v"(a[1]), "=&v"(a[2]), "=&v"(a[3]), "=&v"(b[0]), "=&v"(b[1]), "=&v"(b[2]), "=&v"(b[3])
        : "v"(p[0]), "v"(p[1]), "v"(p[2]), "v"(p[3]), "v"(p[4]), "v"(p[5]), "v"(p[6]), "v"(p[7]), "v"(s[0]), "v"(s[1]),
          "v"(s[2]), "v"(s[3]));
    *hi = u32x4{a[0], a[1], a[2], a[3]};
    *lo = u32x4{b[0], b[1], b[2], b[3]};
}
// The scales (two a word) of 2^(k - 4) to 2^(k + 1), for k = 15 all from 2^11 on (NaN too); zeros for the others.
__device__ __forceinline__ u32x4 large_scales(const u32x4& s, int k) {
    auto in = [k](uint32_t half) { return (half >> 10 & 31u) - (uint32_t)(k + 11) < (k == 15 ? 6u : 5u); };
    u32x4 r;
#pragma unroll
    for (int e = 0; e < 4; ++e) r[e] = (in(s[e]) ? s[e] & 0xFFFFu : 0u) | (in(s[e] >> 16) ? s[e] & 0xFFFF0000u : 0u);
    return r;
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
    p->sh = Kv4Shape{(int)n_slots, nk, 1, (int)(max_pages * page_tokens), (int)rows};
    return SX8_OK;
}

// Row pointers (null: only without rows): 16-byte aligned, strides multiples of 8.
int32_t check_rows(const char* what, const char* name, const void* ptr, int64_t ts, int64_t hs, int64_t rows) {
    if (!ptr && rows > 0) return fail(SX8_ERR_INVALID, "%s: null pointer", what);
    if (!aligned(ptr, 16) || ts % 8 || hs % 8 || ts < 0 || hs < 0 || ts > (int64_t)1 << 40 || hs > (int64_t)1 << 40)
        return fail(SX8_ERR_INVALID, "%s: %s must be 16-byte aligned with strides that are multiples of 8", what, name);
    return SX8_OK;
}

// Output rows of `heads` heads: no two of them share memory.
int32_t check_apart(const char* what, const char* name, int64_t ts, int64_t hs, int64_t rows, int64_t heads, int64_t hd) {
    if (rows == 0 || rows_apart(ts, hs, rows, heads, hd)) return SX8_OK;
    return fail(SX8_ERR_INVALID, "%s: rows of %s overlap", what, name);
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
