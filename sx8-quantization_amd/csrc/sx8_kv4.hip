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
__device__ __forceinline__ int64_t block_offset(const Kv4Pool& p, int slot, int head, int b, int bb) {
    const int at = b >> p.bpp_log2;
    if (b < 0 || at >= p.max_pages) return -1;
    const int page = p.table[(int64_t)slot * p.max_pages + at];
    if (page < 0 || page >= p.n_pages) return -1;
    return page * p.page_bytes + (((int64_t)head << p.bpp_log2) + (b & ((1 << p.bpp_log2) - 1))) * bb;
}

// ---- append ------------------------------------------------------------------------------------
// A work-group encodes the new rows of one block of one head, so that no word of the cache has two writers.
// Eight lanes hold a group of 64 values (16 bytes each): minimum and maximum by three lane exchanges, then each
// lane's eight levels.  K's eight levels of a lane are one word; V's word holds eight tokens of a dimension, so V's
// levels meet in LDS, and a word with tokens of earlier calls keeps their bits.
// 13081 rows of 8 heads of 128 take 20 us (69 MB, 3.5 TB/s; the VALU is busy 56% of the time, 1.7 rounds of work-groups), a
// row of each of 64 slots 4.8, where the chain of lengths, table and rows is all there is.
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
    constexpr int kBB = kv4_block_bytes(HD), CPR = HD / 8, NI = 32 * CPR / 256;   // chunks of a row; rounds of K or V
    __shared__ __align__(8) uint8_t lv[32][HD + 8];
    int64_t* const pre = reinterpret_cast<int64_t*>(dyn_lds);
    Touched t;
    if (!find_touched(p, blockIdx.x, pre, &t)) return;
    const int head = blockIdx.y, tid = threadIdx.x;
    const int64_t off = block_offset(p, t.slot, head, t.block, kBB);
    const int nt = t.t1 - t.t0;
    // every row of the block's share is requested before the first is encoded (and while the page number is on its way)
    constexpr int kStep = 256 / CPR;                                // rows between a thread's chunks
    u32x4 raw[2][NI];
    {
        const uint16_t* const k = in.k + t.row0 * in.k_ts + head * in.k_hs + ((uint32_t)tid / CPR * in.k_ts + tid % CPR * 8);
        const uint16_t* const v = in.v + t.row0 * in.v_ts + head * in.v_hs + ((uint32_t)tid / CPR * in.v_ts + tid % CPR * 8);
#pragma unroll
        for (int i = 0; i < NI; ++i)
            if (tid + 256 * i < nt * CPR) {
                raw[0][i] = *reinterpret_cast<const u32x4*>(k + i * (kStep * in.k_ts));
                raw[1][i] = *reinterpret_cast<const u32x4*>(v + i * (kStep * in.v_ts));
            }
    }
    if (off < 0) return;                                            // (uniform)
    uint8_t* const blk = const_cast<uint8_t*>(p.pages) + off;
#pragma unroll
    for (int which = 0; which < 2; ++which)
#pragma unroll
        for (int i = 0; i < NI; ++i) {
            const int ch = tid + 256 * i;
            if (ch >= nt * CPR) break;                              // (eight lanes of a group alike: CPR is a multiple of 8)
            const int tok = t.t0 + ch / CPR, d0 = ch % CPR * 8, g = d0 / kKv4Group;
            __builtin_assume(tok >= 0 && tok < 32);
            Enc en;
            encode_group<kBf16>(raw[which][i], en);
            // (the low 22 bits of lv are the level)
            if (which == 0) {
                const uint32_t even = en.lv[0] | en.lv[2] << 4 | en.lv[4] << 8 | en.lv[6] << 12;
                const uint32_t odd = en.lv[1] | en.lv[3] << 4 | en.lv[5] << 8 | en.lv[7] << 12;
                *reinterpret_cast<uint32_t*>(blk + kv4_k_word(HD, tok, d0)) = __builtin_amdgcn_perm(odd, even, 0x05040100u);
            } else {
                u32x2 bytes;
#pragma unroll
                for (int w = 0; w < 2; ++w)
                    bytes[w] = __builtin_amdgcn_perm(en.lv[4 * w + 1], en.lv[4 * w], 0x0C0C0400u) |
                               __builtin_amdgcn_perm(en.lv[4 * w + 3], en.lv[4 * w + 2], 0x04000C0Cu);
                *reinterpret_cast<u32x2*>(&lv[tok][d0]) = bytes;
            }
            if (tid % 8 == 0) {
                *reinterpret_cast<uint16_t*>(blk + kv4_param(HD, 2 * which, tok, g)) = (uint16_t)st16<false>(en.s);
                *reinterpret_cast<uint16_t*>(blk + kv4_param(HD, 2 * which + 1, tok, g)) = (uint16_t)st16<false>(en.m);
            }
        }
    __syncthreads();
    // words of four dimensions d0 .. d0 + 3: tokens 4 h + r and 16 + 4 h + r
    for (int i = tid; i < HD; i += 256) {
        const int h = i / (HD / 4), d0 = i % (HD / 4) * 4;
        uint32_t b[8], fresh = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const int tok = e / 4 * 16 + 4 * h + e % 4;
            b[e] = *reinterpret_cast<const uint32_t*>(&lv[tok][d0]) & 0x0F0F0F0Fu;     // (old tokens' bytes were never set)
            if (tok >= t.t0 && tok < t.t1) fresh |= 15u << kv4_shift(e);
        }
        if (fresh == 0) continue;
        // bytes of four dimensions with the levels of two tokens each; byte j of a word is byte d of c[j]
        const uint32_t c[4] = {b[0] | b[2] << 4, b[4] | b[6] << 4, b[1] | b[3] << 4, b[5] | b[7] << 4};
#pragma unroll
        for (int d = 0; d < 4; ++d) {
            const uint32_t word = __builtin_amdgcn_perm(__builtin_amdgcn_perm(c[3], c[2], 0x0C0C0400u + 0x0101u * d),
                                                        __builtin_amdgcn_perm(c[1], c[0], 0x0C0C0400u + 0x0101u * d), 0x05040100u);
            uint32_t* const at = reinterpret_cast<uint32_t*>(blk + kv4_v_word(HD, 4 * h, d0 + d));
            *at = fresh == 0xFFFFFFFFu ? word : (*at & ~fresh) | (word & fresh);
        }
    }
}

// ---- read --------------------------------------------------------------------------------------
// The same cut: a work-group takes one block of one head into LDS (coalesced) and writes its new tokens' rows, K by
// words (eight dimensions of a token), V by four words side by side (eight tokens of four dimensions).  13081 rows of
// 8 heads of 128 in 13.3 us (69 MB, 5.2 TB/s).
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
    for (int i = tid; i < kBB / 16; i += 256)
        reinterpret_cast<u32x4*>(blk)[i] = off < 0 ? u32x4{0u, 0u, 0u, 0u} : reinterpret_cast<const u32x4*>(p.pages + off)[i];
    __syncthreads();
    const int nt = t.t1 - t.t0;
    auto value = [](uint32_t level, float s, float m) { return __builtin_fmaf((float)(int)level, s, m); };
    for (int i = tid; i < nt * CPR; i += 256) {
        const int tok = t.t0 + i / CPR, d0 = i % CPR * 8, g = d0 / kKv4Group;
        const float s = sx8_h2f(*reinterpret_cast<const uint16_t*>(blk + kv4_param(HD, 0, tok, g)));
        const float m = sx8_h2f(*reinterpret_cast<const uint16_t*>(blk + kv4_param(HD, 1, tok, g)));
        const uint32_t word = *reinterpret_cast<const uint32_t*>(blk + kv4_k_word(HD, tok, d0));
        u32x4 w;
#pragma unroll
        for (int e = 0; e < 4; ++e)
            w[e] = pack16<kBf16>(value(word >> kv4_shift(2 * e) & 15u, s, m), value(word >> kv4_shift(2 * e + 1) & 15u, s, m));
        *reinterpret_cast<u32x4*>(out.k + (int64_t)(t.row0 + i / CPR) * out.k_ts + head * out.k_hs + d0) = w;
    }
    for (int i = tid; i < HD; i += 256) {
        const int h = i / (HD / 4), d0 = i % (HD / 4) * 4, g = d0 / kKv4Group;
        uint32_t words[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) words[e] = *reinterpret_cast<const uint32_t*>(blk + kv4_v_word(HD, 4 * h, d0 + e));
        const u32x4 s8 = *reinterpret_cast<const u32x4*>(blk + kv4_param(HD, 2, 4 * h, g));
        const u32x4 m8 = *reinterpret_cast<const u32x4*>(blk + kv4_param(HD, 3, 4 * h, g));
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const int tok = e / 4 * 16 + 4 * h + e % 4;
            if (tok < t.t0 || tok >= t.t1) continue;
            const float s = sx8_h2f(half_of(s8[e >> 1], e)), m = sx8_h2f(half_of(m8[e >> 1], e));
            float x[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) x[k] = value(words[k] >> kv4_shift(e) & 15u, s, m);
            *reinterpret_cast<u32x2*>(out.v + (int64_t)(t.row0 + tok - t.t0) * out.v_ts + head * out.v_hs + d0) =
                u32x2{pack16<kBf16>(x[0], x[1]), pack16<kBf16>(x[2], x[3])};
        }
    }
}

// ---- attend ------------------------------------------------------------------------------------
// The launch's waves share the blocks of all units evenly (sx8_kv4.h) and work apart from each other; a piece is a run
// of blocks of one unit.  Per block a wave computes S^T = K Q^T on v_mfma_f32_16x16x32_f16 with the tokens as
// rows and the unit's 16 query rows as columns, so that a lane (column c, step group h) holds the scores of
// tokens 4 h + r and 16 + 4 h + r of its own query row and the softmax stays in the lane.  The levels go into the
// MFMA as the fp16 subnormals level * 2^-20, which is a shift and a mask for two values and exact; the scale
// multiplies each group's 32-bit sum (q . k = sum_g s_g (q_g . level_g) + m_g sum(q_g)), and the minima's part is
// one more MFMA with sum(q_g) as two fp16 numbers.  O^T += V^T P^T takes the levels in the same way, with p * s of
// each token rounded to two fp16 numbers (22 bits), and the minima's part sum_t p_t m_t,g as MFMAs of their own.
// The MFMA aligns its products by their exponent fields, a subnormal's being 2^-14, and cuts what lies about 25 places below the
// largest: always downwards, so a sum of levels comes out too small by up to half a place a product.  As level * 2^-24 that
// is 2^-16 of a level, which many tokens do not average away while their values do (four slots of up to 131000 tokens: 5.5e-4
// of the outputs); as level * 2^-20 it is 2^-20 of one (1e-5 of them, the plain float32 form 4e-6).
// Query rows are multiplied by a power of two that brings their largest value into [64, 128), which is undone in
// the scale: rows become fp16 within 2^-31 of their largest value (exact where they hold nothing 2^-20 below it, bf16: 2^-23),
// and sum(q_g) fits.
// The running maximum is kept kUp powers of two below the largest score and raised when a score exceeds it by kUp + kSlack,
// so that p is at most 2^13, the largest weight at least 2^10, and p * s holds its 22 bits down to p * s = 2^-3 in those
// units (below that it is within 2^-25).  (Raised at every larger score, four long slots take 54.4 us instead of 51.7.)
// Scales of 2 or more (groups that span 30 or more) would take p * s out of fp16: those go in 2^k times smaller, below 2 and
// from 1/16 on, with their levels 2^k times as large, in matrix products of their own for each of k = 5, 10 and 15 that a
// block has.  So what is kept of a token does not depend on the scales of other groups or tokens.
// Bound by its chain of loads (lengths, table, block) first: a first block takes 6.2 us; then by memory and the VALU together: the
// blocks come at 4.3-5 TB/s, a stream that is only read at 6.1, with the VALU active 55% of the time (four long
// slots).  8 KV heads of 128: 48 slots of 60 .. 8000 tokens 21.7 us and the combine 4.0, 32 slots of 16384 tokens 122-139 us
// by machine.  Three sets of registers ahead instead of two: no faster.
constexpr float kUp = 10.f, kSlack = 3.f;

template <int HD>
constexpr int waves_log2() { return HD == 256 ? 10 : 11; }        // one or two a SIMD of 256 CUs, as registers allow

// Record of a cut unit for the combine; parts == 0: none.  The records lie by unit (slots, heads, tiles) where the host
// knows that there are no more units than waves, so that the combine has a work-group for each; otherwise by the
// wave that has the unit's first block.
struct Kv4Piece {
    int32_t parts, first, tile, head, row0, n, pad[2];      // first: place of its first part
};
static_assert(sizeof(Kv4Piece) == 32, "record");

struct AttendIo {
    const uint16_t* q;
    uint16_t* out;
    int64_t q_ts, q_hs, o_ts, o_hs;
    float scale_log2;
    float* part_o;                        // [2 waves][16][HD]
    float* part_ml;                       // [2 waves][16][2]
    Kv4Piece* piece;                      // [waves]
    int by_unit;
};

constexpr int64_t attend_ws(int64_t hd) {
    return ((int64_t)(2 * 16 * (hd + 2) * 4 + sizeof(Kv4Piece))) << (hd == 256 ? 10 : 11);
}

template <int HD>
struct Kv4Regs {                          // a lane's share of one block
    static constexpr int W = HD / 32, NT = HD / 16, NG = HD / kKv4Group;
    uint32_t kw[2][W], vw[NT];
    u32x4 ks[NG], vs[NG], vm;
    uint32_t km[2][(NG + 1) / 2];
    bool bad;
};

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

// What a wave knows of the slots: with up to 64 of them lane s holds slot s and its place on the line of blocks; with
// more the places lie in LDS.
struct Slots {
    int row0, n, len;
    int64_t end;                          // places of the slots up to this lane's
    int units;                            // (by_unit) units of the slots up to this lane's
};

template <int HD, bool kBf16>
__global__ __launch_bounds__(256, HD == 256 ? 1 : 2) void k_kv4_attend(const Kv4Pool p, const AttendIo io) {
    using Regs = Kv4Regs<HD>;
    constexpr int W = Regs::W, NT = Regs::NT, NG = Regs::NG, kBB = kv4_block_bytes(HD);
    constexpr float kInf = __builtin_inff();
    int64_t* const pre = reinterpret_cast<int64_t*>(dyn_lds);
    const int lane = threadIdx.x & 63, c = lane & 15, h = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + (threadIdx.x >> 6));
    const int S = p.sh.n_slots, G = p.sh.G;
    const bool few = S <= 64;
    Slots sl = {0, 0, 0, 0, 0};
    int32_t* const pre_units = reinterpret_cast<int32_t*>(pre + S + 1);
    int64_t total;
    int units = 0;
    if (few) {
        if (lane < S) {
            kv4_rows(p.sh, p.cu, lane, &sl.row0, &sl.n);
            sl.len = kv4_len(p.sh, p.lens, lane);
            sl.end = kv4_slot_places(p.sh.nk, G, sl.n, sl.len);
            sl.units = p.sh.nk * kv4_tiles(sl.n, G);
        }
        sl.end = wave_prefix(sl.end);
        total = lane_of(sl.end, 63);
        if (io.by_unit) {
            sl.units = (int)wave_prefix(sl.units);
            units = __builtin_amdgcn_readlane(sl.units, 63);
        }
    } else {
        prefix_sums<256>(S, pre, [&](int s) { return kv4_slot_places(p.sh, p.lens, p.cu, s); });
        if (io.by_unit)
            prefix_sums<256>(S, pre_units, [&](int s) {
                int first, n;
                kv4_rows(p.sh, p.cu, s, &first, &n);
                return (int64_t)p.sh.nk * kv4_tiles(n, G);
            });
        __syncthreads();
        total = uniform(pre[S]);
        if (io.by_unit) units = __builtin_amdgcn_readfirstlane(pre_units[S]);
    }
    const int64_t share = kv4_share(total, waves_log2<HD>());
    const int64_t x0 = wave * share, x1 = x0 + share < total ? x0 + share : total;
    int slot = 0;
    if (x0 < total) {
        if (few) slot = __builtin_popcountll(__builtin_amdgcn_ballot_w64(lane < S && sl.end <= x0));
        else
            for (int s = lane; s - lane < S; s += 64) slot += __builtin_popcountll(__builtin_amdgcn_ballot_w64(s < S && pre[s < S ? s + 1 : S] <= x0));
    }
    if ((!io.by_unit || wave >= units) && lane == 0) io.piece[wave].parts = 0;
    for (int64_t x = x0; x < x1;) {
        int row0, n, len;
        int64_t begin;
        int unit0 = 0;
        if (few) {
            while (x >= lane_of(sl.end, slot)) ++slot;
            row0 = __builtin_amdgcn_readlane(sl.row0, slot);
            n = __builtin_amdgcn_readlane(sl.n, slot);
            len = __builtin_amdgcn_readlane(sl.len, slot);
            begin = slot ? lane_of(sl.end, slot - 1) : 0;
            if (io.by_unit) unit0 = slot ? __builtin_amdgcn_readlane(sl.units, slot - 1) : 0;
        } else {
            while (x >= uniform(pre[slot + 1])) ++slot;
            kv4_rows(p.sh, p.cu, slot, &row0, &n);
            row0 = __builtin_amdgcn_readfirstlane(row0);
            n = __builtin_amdgcn_readfirstlane(n);
            len = __builtin_amdgcn_readfirstlane(kv4_len(p.sh, p.lens, slot));
            begin = uniform(pre[slot]);
            if (io.by_unit) unit0 = __builtin_amdgcn_readfirstlane(pre_units[slot]);
        }
        const int nb = kv4_unit_blocks(len), tiles = kv4_tiles(n, G);
        const Kv4Run run = kv4_run(x, x - begin, x1, nb);
        const int b0 = run.b0, bend = run.b1;
        const int64_t here = x;
        x += run.places;
        if (b0 == bend) continue;
        const int head = (int)kv4_div(run.unit, tiles), tile = (int)(run.unit - (int64_t)head * tiles);
        // the column's query row, and the last position it may attend
        const int r = 16 * tile + c, tok = r / G;
        const bool row_ok = tok < n;
        const int lim = row_ok ? len - n + tok : len - 1;
        const int tok_min = 16 * tile / G, tok_max = (16 * tile + 15) / G;
        const int lim_min = len - n + tok_min, lim_max = len - n + (tok_max < n ? tok_max : n - 1);
        const int b1 = lim_max < 0 ? b0 : bend < lim_max / 32 + 1 ? bend : lim_max / 32 + 1;   // blocks it reads
        const int cnt = b1 > b0 ? b1 - b0 : 0;
        int pages = -1;                                                    // lane i: page of block b0 + i0 + i
        auto load_pages = [&](int i0) {
            const int b = b0 + i0 + lane;
            pages = b < b1 ? p.table[(int64_t)slot * p.max_pages + (b >> p.bpp_log2)] : -1;
        };
        auto load = [&](Regs& rg, int i) __attribute__((always_inline)) {
            if (i != 0 && (i & 63) == 0) load_pages(i);
            const int b = b0 + i;
            int page = __builtin_amdgcn_readlane(pages, i & 63);
            rg.bad = page < 0 || page >= p.n_pages;
            page = rg.bad ? 0 : page;
            const uint8_t* base = p.pages + page * p.page_bytes
                + (int64_t)((head << p.bpp_log2) + (b & ((1 << p.bpp_log2) - 1))) * kBB;
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
        load_pages(0);
        // query fragment: fp16 with the row's largest value in [64, 128)
        u32x4 raw[W];
        {
            const int tk = row_ok ? tok : 0, hd = head * G + (row_ok ? r - tok * G : 0);
            const uint16_t* qr = io.q + ((int64_t)row0 + tk) * io.q_ts + hd * io.q_hs + 8 * h;
#pragma unroll
            for (int j = 0; j < W; ++j) raw[j] = *reinterpret_cast<const u32x4*>(qr + 32 * j);
        }
        Regs r0, r1;
        if (cnt > 0) load(r0, 0);
        f16x8 qf[W], qm;
        float kscale;
        {
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
        auto step = [&](Regs& rg, int i) __attribute__((always_inline)) {
            const int b = b0 + i;
            const bool mask = b * 32 + 31 > lim_min || rg.bad;     // past a column's last position, or no page
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
                for (int e = 0; e < 4; ++e) sc[4 * a + e] = __builtin_fmaf(s[e], 1048576.f, mt[e]);
            }
            if (mask) {
                asm volatile("");                // (a branch: as selects these would run for every block)
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const int key = b * 32 + (e / 4) * 16 + 4 * h + e % 4;
                    sc[e] = key <= lim && !rg.bad ? sc[e] : -kInf;
                }
            }
            float mx = sc[0];
#pragma unroll
            for (int e = 1; e < 8; ++e) mx = fmaxf(mx, sc[e]);
            mx *= kscale;
            if (__builtin_amdgcn_ballot_w64(mx > m + (kUp + kSlack)) != 0) {
                const float mn = fmaxf(m, max4(mx - kUp));
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
            if (mask) {
                // a token that some column may not attend must not reach it through 0 * NaN: its scale is zero for that
                // column, and its minimum zero where it is no number (the scale, which is none either, still brings the
                // NaN to the columns that attend it, however small its weight)
                asm volatile("");
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const int key = b * 32 + (e / 4) * 16 + 4 * h + e % 4;
                    if (key > lim || rg.bad)
#pragma unroll
                        for (int g = 0; g < NG; ++g) rg.vs[g][e >> 1] &= e & 1 ? 0xFFFFu : 0xFFFF0000u;
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const uint32_t lo = vm[e] & 0x7FFFu, hi = vm[e] >> 16 & 0x7FFFu;
                    vm[e] = (lo >= 0x7C00u ? 0u : vm[e] & 0xFFFFu) | (hi >= 0x7C00u ? 0u : vm[e] & 0xFFFF0000u);
                }
            }
            u32x4 ph, pl;
            constexpr uint32_t kOnes = 0x3C003C00u;
            split8(pv, u32x4{kOnes, kOnes, kOnes, kOnes}, &ph, &pl);
            const f16x8 vm8 = __builtin_bit_cast(f16x8, vm);
            om = mfma16(vm8, __builtin_bit_cast(f16x8, ph), om);
            om = mfma16(vm8, __builtin_bit_cast(f16x8, pl), om);
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
                        u32x4 hi, lo;
                        split8(pv, s, &hi, &lo);
#pragma unroll
                        for (int t = 4 * g; t < 4 * g + 4; ++t) {
                            uint32_t w = rg.vw[t];
                            asm volatile("" : "+v"(w));          // (here, not ahead of the loop: registers)
                            const f16x8 lv = levels(w) * f16x8(up);
                            o[t] = mfma16(lv, __builtin_bit_cast(f16x8, hi), o[t]);
                            o[t] = mfma16(lv, __builtin_bit_cast(f16x8, lo), o[t]);
                        }
                    }
#pragma unroll
                    for (int e = 0; e < 4; ++e) rg.vs[g][e] &= ~((rg.vs[g][e] >> 14 & 0x00010001u) * 0xFFFFu);
                }
            }
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                u32x4 hi, lo;
                split8(pv, rg.vs[g], &hi, &lo);
                const f16x8 h8 = __builtin_bit_cast(f16x8, hi), l8 = __builtin_bit_cast(f16x8, lo);
#pragma unroll
                for (int t = 4 * g; t < 4 * g + 4; ++t) {
                    const f16x8 lv = levels(rg.vw[t]);
                    o[t] = mfma16(lv, h8, o[t]);
                    o[t] = mfma16(lv, l8, o[t]);
                }
            }
        };
        for (int i = 0; i < cnt; i += 2) {
            if (i + 1 < cnt) load(r1, i + 1);
            step(r0, i);
            if (i + 1 >= cnt) break;
            if (i + 2 < cnt) load(r0, i + 2);
            step(r1, i + 1);
        }
        // O = 2^20 (levels) + (the minima's sum of the group, row g of om)
        l = sum4(l);
        const bool whole = b0 == 0 && bend == nb;
        const float f = whole ? (l == 0.f ? 0.f : 1.f / l) : 1.f;
        const int place = 2 * wave + (here == x0 ? 0 : 1);
        const int64_t at = place * (int64_t)16 + c;
        float* const po = io.part_o + at * HD + 4 * h;
        uint16_t* const dst = io.out + ((int64_t)row0 + tok) * io.o_ts + (head * G + (r - tok * G)) * io.o_hs + 4 * h;
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            const float og = __shfl(om[t / 4], c, 64);
            f32x4 v;
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = __builtin_fmaf(o[t][e], 1048576.f, og) * f;
            if (row_ok) {
                if (whole) *reinterpret_cast<u32x2*>(dst + 16 * t) = u32x2{pack16<kBf16>(v[0], v[1]), pack16<kBf16>(v[2], v[3])};
                else *reinterpret_cast<f32x4*>(po + 16 * t) = v;
            }
        }
        if (!whole && h == 0 && row_ok) {
            io.part_ml[at * 2] = m;
            io.part_ml[at * 2 + 1] = l;
        }
        // the unit's record is written by its first piece; a unit that is cut goes on in the next waves
        // (a cu that runs backwards can name more units than rows allow: those have no record)
        const int64_t rec = io.by_unit ? unit0 + run.unit : wave;
        if (b0 == 0 && lane == 0 && (io.by_unit || !whole) && rec < (1 << waves_log2<HD>())) {
            Kv4Piece pc;
            pc.parts = whole ? 0 : kv4_parts(begin + run.unit * (nb + kKv4Begin) + kKv4Begin, nb, share, wave);
            pc.first = place;
            pc.tile = tile;
            pc.head = head;
            pc.row0 = row0;
            pc.n = n;
            io.piece[rec] = pc;
        }
    }
}

// Units that were cut: work-group (i, row) takes a row of record i and adds the unit's parts up in their order (part 0 at its
// place, part j at place 2 (wave + j)).  The parts are shared by kWaves waves, whose sums meet in LDS.  A launch costs 1.8
// us and three dependent loads; 48 slots of up to 8000 tokens take 4.0-4.7 us, 16 slots of 8 new tokens 5.6-6.0 (work-groups of
// 16 waves for four rows at once: 5.9 and 6.5; two waves a row: 4.8 and 5.1, but twice the rounds where one slot of
// many has most of the tokens).
template <int HD, bool kBf16, int kWaves>
__global__ __launch_bounds__(64 * kWaves) void k_kv4_combine(const AttendIo io, int G) {
    constexpr int N = HD / 64, kU = 8;                            // kU: parts requested together
    typedef float vecN __attribute__((ext_vector_type(N)));
    const Kv4Piece pc = io.piece[blockIdx.x];
    const int row = blockIdx.y;
    if (pc.parts == 0 || row >= min(16, pc.n * G - 16 * pc.tile)) return;
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    __shared__ float sml[kWaves][2];
    __shared__ vecN so[kWaves][64];
    auto at = [&](int i) { return (int64_t)(i == 0 ? pc.first : 2 * (pc.first / 2 + i)) * 16 + row; };
    const int per = (pc.parts + kWaves - 1) / kWaves, i0 = w * per, i1 = min(i0 + per, pc.parts);
    float m = -__builtin_inff(), den = 0.f;
    vecN acc = 0.f;
    for (int i = i0; i < i1; i += kU) {
        float pm[kU], pl[kU];
        vecN v[kU];
#pragma unroll
        for (int u = 0; u < kU; ++u) {
            const int64_t a = at(min(i + u, i1 - 1));
            pm[u] = io.part_ml[a * 2];
            pl[u] = io.part_ml[a * 2 + 1];
            v[u] = reinterpret_cast<const vecN*>(io.part_o + a * HD)[lane];
        }
        __builtin_amdgcn_sched_barrier(0);
        float mn = m;
#pragma unroll
        for (int u = 0; u < kU; ++u) mn = fmaxf(mn, pm[u]);
        const float alpha = m == mn ? 1.f : __builtin_amdgcn_exp2f(m - mn);
        m = mn;
        den *= alpha;
        acc *= alpha;
#pragma unroll
        for (int u = 0; u < kU; ++u) {
            if (i + u >= i1) continue;
            const float f = pm[u] == m ? 1.f : __builtin_amdgcn_exp2f(pm[u] - m);
            den = __builtin_fmaf(f, pl[u], den);
            acc = __builtin_elementwise_fma(vecN(f), v[u], acc);
        }
    }
    if (lane == 0) {
        sml[w][0] = m;
        sml[w][1] = den;
    }
    so[w][lane] = acc;
    __syncthreads();
    if (w != 0) return;
    float mm = m;
#pragma unroll
    for (int i = 1; i < kWaves; ++i) mm = fmaxf(mm, sml[i][0]);
    const float f0 = m == mm ? 1.f : __builtin_amdgcn_exp2f(m - mm);
    den *= f0;
    acc *= f0;
#pragma unroll
    for (int i = 1; i < kWaves; ++i) {
        const float f = sml[i][0] == mm ? 1.f : __builtin_amdgcn_exp2f(sml[i][0] - mm);
        den = __builtin_fmaf(f, sml[i][1], den);
        acc = __builtin_elementwise_fma(vecN(f), so[i][lane], acc);
    }
    acc *= den == 0.f ? 0.f : 1.f / den;
    const int rr = 16 * pc.tile + row, tk = rr / G;
    uint16_t* dst = io.out + ((int64_t)pc.row0 + tk) * io.o_ts + (pc.head * G + (rr - tk * G)) * io.o_hs + N * lane;
    if constexpr (N == 1) *dst = (uint16_t)st16<kBf16>(acc[0]);
    else
#pragma unroll
        for (int e = 0; e < N; e += 2) *reinterpret_cast<uint32_t*>(dst + e) = pack16<kBf16>(acc[e], acc[e + 1]);
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
        hipLaunchKernelGGL((k_kv4_append<decltype(d)::value, decltype(b)::value>), grid, dim3(256),
                           cu && n_slots > 64 ? prefix_bytes(p) : 0, as_stream(stream), p, in);
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
    if (rc == SX8_OK) rc = check_apart(what, "k", k_ts, k_hs, rows, nk, hd);
    if (rc == SX8_OK) rc = check_apart(what, "v", v_ts, v_hs, rows, nk, hd);
    if (rc != SX8_OK) return rc;
    if (rows == 0) return ok();
    const RowsOut out{(uint16_t*)k, (uint16_t*)v, k_ts, k_hs, v_ts, v_hs};
    const dim3 grid((unsigned)kv4_touched_most(n_slots, rows, cu != nullptr), (unsigned)nk);
    by_kind(hd, dtype, [&](auto d, auto b) {
        hipLaunchKernelGGL((k_kv4_read<decltype(d)::value, decltype(b)::value>), grid, dim3(256),
                           cu && n_slots > 64 ? prefix_bytes(p) : 0, as_stream(stream), p, out);
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
    rc = check_apart(what, "out", o_ts, o_hs, rows, nh, hd);
    if (rc != SX8_OK) return rc;
    if (!(scale > 0.f) || !(scale < __builtin_inff()))
        return fail(SX8_ERR_INVALID, "%s: scale must be positive and finite", what);
    if (!workspace || workspace_bytes < attend_ws(hd) || !aligned(workspace, 256))
        return fail(SX8_ERR_INVALID, "%s: workspace needs %lld bytes, 256-byte aligned", what, (long long)attend_ws(hd));
    if (rows * (nh / nk) > 0x7FFFFF00) return fail(SX8_ERR_UNSUPPORTED, "%s: over 2^31 query rows of a KV head", what);
    if (rows == 0) return ok();
    p.sh.G = nh / nk;
    const int64_t waves = (int64_t)1 << (hd == 256 ? 10 : 11);
    AttendIo io{(const uint16_t*)q, (uint16_t*)out, q_ts, q_hs, o_ts, o_hs, scale * 1.4426950408889634f, nullptr, nullptr,
                nullptr, 0};
    io.piece = reinterpret_cast<Kv4Piece*>(workspace);
    io.part_o = reinterpret_cast<float*>(io.piece + waves);
    io.part_ml = io.part_o + 2 * waves * 16 * hd;
    // units at most: a slot with n rows has nk ceil(n G / 16) of them
    const int64_t G = p.sh.G, live = n_slots < rows ? n_slots : rows;
    const int64_t units = nk * (cu ? rows * G / 16 + live : n_slots * ((G + 15) / 16));
    io.by_unit = units <= waves;
    const unsigned entries = (unsigned)(io.by_unit ? units : waves), used = (unsigned)(cu ? (rows * G < 16 ? rows * G : 16) : (G < 16 ? G : 16));
    // few rows in all: a row's parts are shared by 16 waves, else by four
    const bool narrow = entries * used <= 512;
    by_kind(hd, dtype, [&](auto d, auto b) {
        constexpr int HD = decltype(d)::value;
        constexpr bool kBf = decltype(b)::value;
        hipLaunchKernelGGL((k_kv4_attend<HD, kBf>), dim3((1 << waves_log2<HD>()) / 4), dim3(256),
                           n_slots <= 64 ? 0 : prefix_bytes(p) * 3 / 2, as_stream(stream), p, io);
        const dim3 grid(entries, used);
        if (narrow) hipLaunchKernelGGL((k_kv4_combine<HD, kBf, 16>), grid, dim3(1024), 0, as_stream(stream), io, p.sh.G);
        else hipLaunchKernelGGL((k_kv4_combine<HD, kBf, 4>), grid, dim3(256), 0, as_stream(stream), io, p.sh.G);
    });
    return check_launch(what);
}
