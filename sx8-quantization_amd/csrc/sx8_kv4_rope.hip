// sx8_kv4_rope.hip -- new rows of the paged 4-bit cache with their norm and rotation on the way (include/sx8_paged.h):
// query rows to memory, K and V rows into the slots' pages.
//
// Per head row x: x <- x / sqrt(mean x^2 + eps) w where weights are given, then the pairs (a, b) of the first `rot`
// dimensions become (a cos - b sin, b cos + a sin) with the row's place in the tables.  All of it in binary64, which costs
// nothing here (the launch waits for memory) and makes the 16-bit values, and with them the levels, those of the exact
// formula: a K value that falls to the other side of a rounding moves the ends of its group or its level.  Rounded once,
// to float32 and from there to 16 bits; K and V are then encoded as sx8_kv4_append does it.
// Bound by memory where rows are many (9761 rows of nine prompts, 32 heads over 8 of 128: 211 MB in 56 us, 3.8 TB/s, and in 44 where the
// rows lie in the last-level cache yet) and by a launch of
// five dependent round trips where they are few (64 rows, one a slot: 6.7 us).
#include "sx8_kv4_core.h"

namespace sx8 {
namespace {

struct RopeIn {
    const void *q, *k, *v;
    int64_t q_ts, q_hs, k_ts, k_hs, v_ts, v_hs;
    uint16_t* out;
    int64_t o_ts, o_hs;
    const float *cos, *sin;
    int64_t table_rows;
    const int32_t* depth;
    int32_t* marks;                         // [n_slots][kMarkWords], or null
    const uint16_t *qw, *kw;
    double eps;
    int rot, heads;                         // heads: query heads of a work-group
};

template <int kIn>                          // 0: fp16, 1: bf16, 2: float32
struct Row {
    using T = uint16_t;
    static __device__ __forceinline__ void load(const T* p, float (&x)[8]) {
        const u32x4 w = *reinterpret_cast<const u32x4*>(p);
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = ld16<kIn == 1>(half_of(w[e >> 1], e));
    }
};
template <>
struct Row<2> {
    using T = float;
    static __device__ __forceinline__ void load(const T* p, float (&x)[8]) {
        const f32x4 a = reinterpret_cast<const f32x4*>(p)[0], b = reinterpret_cast<const f32x4*>(p)[1];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            x[e] = a[e];
            x[4 + e] = b[e];
        }
    }
};

template <bool kBf16>
__device__ __forceinline__ u32x4 pack8(const float (&x)[8]) {
    u32x4 w;
#pragma unroll
    for (int e = 0; e < 4; ++e) w[e] = pack16<kBf16>(x[2 * e], x[2 * e + 1]);
    return w;
}

// Dimensions d0 .. d0 + 7 of a head row (the lanes of a row, HD / 8 of them, come together).
template <int HD, int kIn, bool kBf16, bool kInter>
__device__ __forceinline__ u32x4 turned(const typename Row<kIn>::T* row, int d0, const uint16_t* w, double eps,
                                        const float* cos, const float* sin, int rot) {
    float x[8], y[8];
    Row<kIn>::load(row + d0, x);
    const int half = rot / 2, low = d0 < half;
    const bool turns = d0 < rot;
    const int other = kInter || !turns ? d0 : low ? d0 + half : d0 - half;
    Row<kIn>::load(row + other, y);
    double a[8], b[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        a[e] = x[e];
        b[e] = y[e];
    }
    if (w) {
        double sum = 0.0;
#pragma unroll
        for (int e = 0; e < 8; ++e) sum = __builtin_fma(a[e], a[e], sum);
#pragma unroll
        for (int o = 1; o < HD / 8; o <<= 1) sum += __shfl_xor(sum, o, 64);
        const double inv = 1.0 / sqrt(sum / HD + eps);
        float wa[8], wb[8];
        Row<kBf16>::load(w + d0, wa);
        Row<kBf16>::load(w + other, wb);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            a[e] = a[e] * inv * wa[e];
            b[e] = b[e] * inv * wb[e];
        }
    }
    float r[8];
    if (!turns) {
#pragma unroll
        for (int e = 0; e < 8; ++e) r[e] = (float)a[e];
    } else if constexpr (kInter) {
        const f32x4 c = *reinterpret_cast<const f32x4*>(cos + d0 / 2), s = *reinterpret_cast<const f32x4*>(sin + d0 / 2);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            r[2 * e] = (float)(a[2 * e] * c[e] - a[2 * e + 1] * s[e]);
            r[2 * e + 1] = (float)(a[2 * e + 1] * c[e] + a[2 * e] * s[e]);
        }
    } else {
        const int at = low ? d0 : d0 - half;
        float c[8], s[8];
        Row<2>::load(cos + at, c);
        Row<2>::load(sin + at, s);
#pragma unroll
        for (int e = 0; e < 8; ++e) r[e] = (float)(a[e] * c[e] + b[e] * (low ? -(double)s[e] : (double)s[e]));
    }
    return pack8<kBf16>(r);
}

// Work-groups (block, y): y < nk encodes the K and V rows of a head, the others turn the rows of `heads` of
// the query heads that share one.
template <int HD, int kIn, bool kBf16, bool kInter, bool kOne>       // kOne: one query head
__global__ __launch_bounds__(256) void k_kv4_append_rope(const Kv4Pool p, const RopeIn in) {
    using T = typename Row<kIn>::T;
    constexpr int kBB = kv4_block_bytes(HD), CPR = HD / 8;
    __shared__ __align__(8) uint8_t lv[32][HD + 8];
    __shared__ int place[32];               // of a token in the tables, -1: outside
    int64_t* const pre = reinterpret_cast<int64_t*>(dyn_lds);
    // The slot's mark, asked for with the lengths that say which slot it is, and only where pages are written (9761 rows of nine
    // prompts and their read 52.3 us, without marks 51.9, looked at by all work-groups 53.0).
    const bool looks = in.marks && (int)blockIdx.y < p.sh.nk, late = p.cu && p.sh.n_slots > 64;
    int mark = 0;
    if (looks && !late) mark = in.marks[kMarkWords * (p.cu ? min((int)threadIdx.x & 63, p.sh.n_slots - 1) : (int)blockIdx.x)];
    Touched t;
    if (!find_touched(p, blockIdx.x, pre, &t)) return;
    if (looks && p.cu) mark = late ? in.marks[kMarkWords * t.slot] : __builtin_amdgcn_readlane(mark, t.slot);
    const int head = blockIdx.y, tid = threadIdx.x, nt = t.t1 - t.t0, half = in.rot / 2;
    // (the last tokens of a slot that was refused its new ones are older: nothing of it may be overwritten)
    const bool refused = mark < 0;
    if (tid < nt) {
        const int64_t at = in.depth ? (int64_t)t.first + in.depth[t.row0 + tid] : (int64_t)t.block * 32 + t.t0 + tid;
        const bool inside = at >= 0 && at < in.table_rows;
        place[t.t0 + tid] = !refused && inside ? (int)at : -1;
        if (in.marks && !inside && head == 0) {                      // (a row that stays out of the pages)
            int32_t* const of = in.marks + kMarkWords * t.slot;
            const int row = t.block * 32 + t.t0 + tid - t.first;
            if (row < kMarkRows) atomicOr(&of[1 + row / 32], 1 << row % 32);
            atomicMin(of, row < kMarkRows ? kMarkSome : row);
        }
    }
    __syncthreads();
    if (head >= p.sh.nk) {
        const int G = p.sh.G, hs = kOne ? 1 : in.heads, cuts = (G + hs - 1) / hs, y = head - p.sh.nk, h0 = kOne ? 0 : y % cuts * hs;
        const int h = kOne ? y : y / cuts * G + h0, per = kOne ? 1 : min(hs, G - h0);
        const T* const q = static_cast<const T*>(in.q) + t.row0 * in.q_ts + h * in.q_hs;
        uint16_t* const out = in.out + t.row0 * in.o_ts + h * in.o_hs;
        for (int ch = tid; ch < nt * per * CPR; ch += 256) {
            const int hr = ch / CPR, i = kOne ? hr : hr / per, g = kOne ? 0 : hr - i * per, d0 = ch % CPR * 8, at = place[t.t0 + i];
            u32x4 r = {0u, 0u, 0u, 0u};
            if (at >= 0)
                r = turned<HD, kIn, kBf16, kInter>(q + i * in.q_ts + g * in.q_hs, d0, in.qw, in.eps, in.cos + (int64_t)at * half,
                                                   in.sin + (int64_t)at * half, in.rot);
            *reinterpret_cast<u32x4*>(out + i * in.o_ts + g * in.o_hs + d0) = r;
        }
        return;
    }
    const int64_t off = block_offset(p, t.slot, head, t.block, kBB);
    if (off < 0) return;                                            // (uniform)
    uint8_t* const blk = const_cast<uint8_t*>(p.pages) + off;
    const T* const k = static_cast<const T*>(in.k) + t.row0 * in.k_ts + head * in.k_hs;
    const T* const v = static_cast<const T*>(in.v) + t.row0 * in.v_ts + head * in.v_hs;
    for (int ch = tid; ch < nt * CPR; ch += 256) {
        const int i = ch / CPR, tok = t.t0 + i, d0 = ch % CPR * 8, g = d0 / kKv4Group, at = place[tok];
        __builtin_assume(tok >= 0 && tok < 32);
        if (at < 0) continue;                                       // (a row's lanes alike)
        Enc en;
        encode_group<kBf16>(turned<HD, kIn, kBf16, kInter>(k + i * in.k_ts, d0, in.kw, in.eps, in.cos + (int64_t)at * half,
                                                           in.sin + (int64_t)at * half, in.rot), en);
        // (the low 22 bits of lv are the level)
        const uint32_t even = en.lv[0] | en.lv[2] << 4 | en.lv[4] << 8 | en.lv[6] << 12;
        const uint32_t odd = en.lv[1] | en.lv[3] << 4 | en.lv[5] << 8 | en.lv[7] << 12;
        *reinterpret_cast<uint32_t*>(blk + kv4_k_word(HD, tok, d0)) = __builtin_amdgcn_perm(odd, even, 0x05040100u);
        if (tid % 8 == 0) {
            *reinterpret_cast<uint16_t*>(blk + kv4_param(HD, 0, tok, g)) = (uint16_t)st16<false>(en.s);
            *reinterpret_cast<uint16_t*>(blk + kv4_param(HD, 1, tok, g)) = (uint16_t)st16<false>(en.m);
        }
        u32x4 raw;
        if constexpr (kIn == 2) {
            float x[8];
            Row<kIn>::load(v + i * in.v_ts + d0, x);
            raw = pack8<kBf16>(x);
        } else {
            raw = *reinterpret_cast<const u32x4*>(v + i * in.v_ts + d0);
        }
        encode_group<kBf16>(raw, en);
        u32x2 bytes;
#pragma unroll
        for (int w = 0; w < 2; ++w)
            bytes[w] = __builtin_amdgcn_perm(en.lv[4 * w + 1], en.lv[4 * w], 0x0C0C0400u) |
                       __builtin_amdgcn_perm(en.lv[4 * w + 3], en.lv[4 * w + 2], 0x04000C0Cu);
        *reinterpret_cast<u32x2*>(&lv[tok][d0]) = bytes;
        if (tid % 8 == 0) {
            *reinterpret_cast<uint16_t*>(blk + kv4_param(HD, 2, tok, g)) = (uint16_t)st16<false>(en.s);
            *reinterpret_cast<uint16_t*>(blk + kv4_param(HD, 3, tok, g)) = (uint16_t)st16<false>(en.m);
        }
    }
    __syncthreads();
    // V's words of four dimensions d0 .. d0 + 3: tokens 4 h + r and 16 + 4 h + r (as k_kv4_append writes them)
    for (int i = tid; i < HD; i += 256) {
        const int h = i / (HD / 4), d0 = i % (HD / 4) * 4;
        uint32_t b[8], fresh = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const int tok = e / 4 * 16 + 4 * h + e % 4;
            b[e] = *reinterpret_cast<const uint32_t*>(&lv[tok][d0]) & 0x0F0F0F0Fu;
            if (tok >= t.t0 && tok < t.t1 && place[tok] >= 0) fresh |= 15u << kv4_shift(e);
        }
        if (fresh == 0) continue;
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

}  // namespace
}  // namespace sx8

extern "C" int32_t sx8_kv4_append_rope(uint8_t* pages, const int32_t* table, const int32_t* lens, const int32_t* cu,
                                       int64_t n_slots, int64_t max_pages, int64_t n_pages, const void* q, const void* k,
                                       const void* v, void* out, int64_t rows, int64_t q_ts, int64_t q_hs, int64_t k_ts,
                                       int64_t k_hs, int64_t v_ts, int64_t v_hs, int64_t o_ts, int64_t o_hs, int32_t nh,
                                       int32_t nk, int32_t hd, int32_t page_tokens, const float* cos_t, const float* sin_t,
                                       int64_t table_rows, int32_t rot, int32_t interleaved, const int32_t* depth,
                                       const void* q_norm, const void* k_norm, double eps, int32_t in_dtype, int32_t dtype,
                                       void* stream) {
    return sx8_kv4_append_rope_marked(pages, table, lens, cu, n_slots, max_pages, n_pages, q, k, v, out, rows, q_ts, q_hs, k_ts,
                                      k_hs, v_ts, v_hs, o_ts, o_hs, nh, nk, hd, page_tokens, cos_t, sin_t, table_rows, rot,
                                      interleaved, depth, nullptr, q_norm, k_norm, eps, in_dtype, dtype, stream);
}

extern "C" int32_t sx8_kv4_append_rope_marked(uint8_t* pages, const int32_t* table, const int32_t* lens, const int32_t* cu,
                                              int64_t n_slots, int64_t max_pages, int64_t n_pages, const void* q, const void* k,
                                              const void* v, void* out, int64_t rows, int64_t q_ts, int64_t q_hs, int64_t k_ts,
                                              int64_t k_hs, int64_t v_ts, int64_t v_hs, int64_t o_ts, int64_t o_hs, int32_t nh,
                                              int32_t nk, int32_t hd, int32_t page_tokens, const float* cos_t,
                                              const float* sin_t, int64_t table_rows, int32_t rot, int32_t interleaved,
                                              const int32_t* depth, int32_t* marks, const void* q_norm, const void* k_norm,
                                              double eps, int32_t in_dtype, int32_t dtype, void* stream) {
    using namespace sx8;
    const char* what = "sx8_kv4_append_rope";
    Kv4Pool p;
    int32_t rc = make_pool(what, &p, pages, table, lens, cu, n_slots, max_pages, n_pages, rows, nk, hd, page_tokens, dtype);
    if (rc == SX8_OK) rc = check_rows(what, "q", q, q_ts, q_hs, rows);
    if (rc == SX8_OK) rc = check_rows(what, "k", k, k_ts, k_hs, rows);
    if (rc == SX8_OK) rc = check_rows(what, "v", v, v_ts, v_hs, rows);
    if (rc == SX8_OK) rc = check_rows(what, "out", out, o_ts, o_hs, rows);
    if (rc != SX8_OK) return rc;
    if (nh <= 0 || nh % nk || nh / nk > 256 || nh + nk > 65535)
        return fail(SX8_ERR_INVALID, "%s: nh must be a multiple of nk, at most 256 nk (and 65535 - nk)", what);
    rc = check_apart(what, "out", o_ts, o_hs, rows, nh, hd);
    if (rc != SX8_OK) return rc;
    if (in_dtype != 2 && in_dtype != dtype)
        return fail(SX8_ERR_INVALID, "%s: rows must be of dtype or float32 (in_dtype 2)", what);
    if (!cos_t || !sin_t || !aligned(cos_t, 16) || !aligned(sin_t, 16) || table_rows <= 0 || table_rows > 0x7FFFFFFF)
        return fail(SX8_ERR_INVALID, "%s: cos and sin must be tables of 1..2^31 - 1 rows, 16-byte aligned", what);
    if (rot < 16 || rot > hd || rot % 16) return fail(SX8_ERR_INVALID, "%s: rot must be a multiple of 16 up to hd", what);
    if (!aligned(depth, 4) || !aligned(marks, 4) || !aligned(q_norm, 16) || !aligned(k_norm, 16))
        return fail(SX8_ERR_INVALID, "%s: depth and marks must be 4-byte aligned, q_norm and k_norm 16-byte", what);
    if (!(eps >= 0.0) || !(eps < __builtin_inff())) return fail(SX8_ERR_INVALID, "%s: eps must not be negative", what);
    if (out == q && rows > 0) return fail(SX8_ERR_INVALID, "%s: out may not be q", what);
    if (rows == 0) return ok();
    p.sh.G = nh / nk;
    // A thread turns eight values a round; a work-group takes as many query heads as its 256 threads have rows for (64 rows of
    // 32 heads of 128, one a slot: 6.7 us with four heads, 9.7 with one; 9761 rows of nine prompts: 48 and 44).
    const int64_t in_block = cu ? (rows + n_slots - 1) / n_slots : 1;
    const int fit = (int)(256 / ((in_block < 32 ? in_block : 32) * (hd / 8))), heads = fit < 1 ? 1 : fit > p.sh.G ? p.sh.G : fit;
    const RopeIn in{q, k, v, q_ts, q_hs, k_ts, k_hs, v_ts, v_hs, (uint16_t*)out, o_ts, o_hs, cos_t, sin_t, table_rows, depth, marks,
                    (const uint16_t*)q_norm, (const uint16_t*)k_norm, eps, rot, heads};
    const dim3 grid((unsigned)kv4_touched_most(n_slots, rows, cu != nullptr), (unsigned)(nk + nk * ((p.sh.G + heads - 1) / heads)));
    by_kind(hd, dtype, [&](auto d, auto b) {
        constexpr int HD = decltype(d)::value;
        constexpr bool kBf = decltype(b)::value;
        auto go = [&](auto kernel) {
            hipLaunchKernelGGL(kernel, grid, dim3(256), cu && n_slots > 64 ? prefix_bytes(p) : 0, as_stream(stream), p, in);
        };
        auto of = [&](auto in_kind, auto inter) {
            constexpr int kIn = decltype(in_kind)::value;
            constexpr bool kInter = decltype(inter)::value;
            if (heads == 1) go(k_kv4_append_rope<HD, kIn, kBf, kInter, true>);
            else go(k_kv4_append_rope<HD, kIn, kBf, kInter, false>);
        };
        auto kind = [&](auto in_kind) {
            if (interleaved) of(in_kind, std::true_type{});
            else of(in_kind, std::false_type{});
        };
        if (in_dtype == 2) kind(std::integral_constant<int, 2>{});
        else kind(std::integral_constant<int, kBf>{});
    });
    return check_launch(what);
}
