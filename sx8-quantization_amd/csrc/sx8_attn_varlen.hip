// sx8_attn_varlen.hip -- attention of packed sequences (include/sx8_paged.h: sx8_attn_varlen).
#include <type_traits>

#include "sx8_buffer.h"
#include "sx8_host.h"
#include "sx8_kv4_dev.h"
#include "sx8_paged.h"

namespace sx8 {
namespace {

// A work-group takes 128 query rows of one head of a sequence, 32 to each of its four waves, and walks the keys in
// tiles that all waves read from LDS.  Per 32 keys a wave computes S^T = K Q^T on the 32x32x16 MFMA with the keys as
// rows and its queries as columns, so that lane 32 h + c holds scores of query c alone (keys 8 (r / 4) + 4 h + r % 4 in
// accumulator r) and the online softmax needs one exchange, with lane ^ 32.  O^T += V^T P^T takes P^T from those
// accumulators as they lie (the order of the contracted keys is free: slot t of half h of step st is key
// 16 st + 8 (t / 4) + 4 h + t % 4), and V^T by the LDS transpose read, which hands a lane four keys of its dimension.
// K and V go from memory to LDS directly, the next tile while this one is computed; rows past the sequence's
// last key lie past the buffer and come as zeros.  A 16-byte chunk of a row lies at its position XOR a few bits of
// the row, so that neither kind of read meets bank conflicts (the swap is made in the load's address).
// Bound by the matrix cores and the softmax's VALU, which two waves a SIMD of different work-groups overlap: one prompt of
// 8192 tokens (32 heads over 8 of 128, bf16) takes 515-550 us by machine, 1000-1067 TFLOP/s, where a library product of
// 8192^3 reaches 1100-1150: the MFMA is busy 51% of a SIMD's cycles and the VALU 46%.  Short prompts are bound by a
// work-group's start (about 5 us: lengths, query, first tile): 24 of
// 40 .. 2000 tokens 230 us, three of up to 96 tokens 7.  s_setprio around the products (541 us against 533), tiles of 32
// keys with three waves a SIMD (544 against 528) and work-groups that stay and request the next rows ahead (561 against
// 515) were slower.  Heads of 256 leave room for one wave a SIMD: 8192 tokens of 16 heads over 4 take 699 us (787 TFLOP/s;
// tiles of 32 keys 719); the next tile's scores computed beside this one's softmax 767 (881 with tiles of 32).
template <int HD>
struct VarTile {
    static constexpr int kKeys = 64;                         // of a tile
    static constexpr int kChunks = HD / 8;                   // 16-byte chunks of a row
    static constexpr int kBytes = kKeys * HD * 2;            // of K or V
    __device__ static int k_swz(int row) { return row & (HD == 128 ? 15 : 7); }
    __device__ static int v_swz(int row) { return HD == 64 ? (row >> 1 & 1) << 2 : (row & 3) << 2; }
};

struct VarIo {
    const uint16_t* q;
    const uint16_t* k;
    const uint16_t* v;
    uint16_t* out;
    const int32_t* cu_q;
    const int32_t* cu_k;
    int64_t q_ts, q_hs, k_ts, k_hs, v_ts, v_hs, o_ts, o_hs;
    int Tq, Tk, n_seq, nh, nk;
    float scale_log2;
    // keys in `splits` parts (gridDim.y): per work-group (x, y) 128 rows of sums and their (maximum, sum of weights)
    int splits;
    float* part_o;                        // [x][y][128][HD]
    float* part_ml;                       // [x][y][128][2]
    struct VarRecord* record;             // [x]
};
struct VarRecord {                        // rows that the parts of x are for; n == 0: none
    int32_t q_first, q0, n, head;
};

constexpr int kRows = 128;

// Rows of sequence b in a packed tensor of T rows: first row and count.
__device__ __forceinline__ void seq_rows(const int32_t* cu, int T, int b, int* first, int* n) {
    const int a = kv4_clamp(cu[b], 0, T), e = kv4_clamp(cu[b + 1], a, T);
    *first = a;
    *n = e - a;
}

typedef __attribute__((address_space(3))) unsigned char lds_u8;

// A raw buffer over `bytes` bytes at p (as make_rsrc), in scalar registers for load_lds.  A memory access may read a scalar
// register that the VALU wrote five states later, which the compiler does not see to in an asm block: the wait is here.
__device__ __forceinline__ u32x4 scalar_rsrc(const void* p, uint32_t bytes) {
    const uint64_t a = reinterpret_cast<uint64_t>(p);
    u32x4 r = {(uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)a),
               (uint32_t)__builtin_amdgcn_readfirstlane((int)((uint32_t)(a >> 32) & 0xFFFFu)),
               (uint32_t)__builtin_amdgcn_readfirstlane((int)bytes), (uint32_t)kRsrcFlags};
    asm volatile("s_nop 4" : "+s"(r));
    return r;
}
// 16 bytes a lane from the buffer to the 1 KB of LDS at byte `dst`; no register is written, and the kernel waits for
// vmcnt(0) and a barrier before it reads that LDS.  The builtin does the same, but the compiler then waits for it before
// every LDS read that might be of the same place, which is every one (prompt of 8192: 730 us against 603).
__device__ __forceinline__ void load_lds(const u32x4& r, int dst, int off) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(dst), "v"(off), "s"(r)
                 : "memory", "m0");
}
// Lane i of 16 names the eight bytes of key i / 4 that hold dimensions 4 (i % 4) .. + 3, and gets dimension i of the four keys.
__device__ __forceinline__ u32x2 read_tr(const unsigned char* at) {
    typedef short s16x4 __attribute__((ext_vector_type(4)));
    return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)at));
}

template <bool kBf16>
struct Mma;
template <>
struct Mma<false> {
    typedef _Float16 vec8 __attribute__((ext_vector_type(8)));
    template <typename A>
    __device__ static A mul(u32x4 a, u32x4 b, A c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(vec8, a), __builtin_bit_cast(vec8, b), c, 0, 0, 0);
    }
};
template <>
struct Mma<true> {
    typedef __bf16 vec8 __attribute__((ext_vector_type(8)));
    template <typename A>
    __device__ static A mul(u32x4 a, u32x4 b, A c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(vec8, a), __builtin_bit_cast(vec8, b), c, 0, 0, 0);
    }
};

// K and V of two tiles, and before that the prefix sums of the sequences' tiles
template <int HD>
constexpr int var_lds_bytes() {
    constexpr int a = 4 * VarTile<HD>::kBytes, b = (kKv4MaxSlots + 1) * 8;
    return a > b ? a : (b + 15) / 16 * 16;
}

// A wave's rows key by key, over the keys that each attends alone: for rows in whose sums there is a value that is no
// finite number (2 to 5 us a key: 8192 tokens of 32 heads take 18 ms with a NaN in one of the last keys' values, 41 with one in
// the first's).  Such a value reaches the row however small its weight: one that underflows counts as 1
// there, and a sum that is not finite is not scaled.  Lane 32 h + c holds the row c's dimensions 32 n + 8 g + 4 h + r, as the
// accumulators do.
template <int HD, bool kBf16, typename V, int NT>
__device__ __forceinline__ void slow_rows(const uint16_t* q, const uint16_t* k, const uint16_t* v, const VarIo& io,
                                          int from, int to, int lim, int h, V (&o)[NT], float& m, float& l) {
    m = -__builtin_inff();
    l = 0.f;
#pragma unroll
    for (int n = 0; n < NT; ++n) o[n] = 0.f;
    for (int key = from; key < to; ++key) {
        float s = 0.f;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int d = 32 * n + 8 * (r >> 2) + 4 * h + (r & 3);
                s = __builtin_fmaf(ld16<kBf16>(q[d]), ld16<kBf16>(k[key * io.k_ts + d]), s);
            }
        s = (s + __shfl_xor(s, 32, 64)) * io.scale_log2;
        if (key > lim) continue;
        const float mn = fmaxf(m, s), alpha = m == mn ? 1.f : __builtin_amdgcn_exp2f(m - mn);
        const float p = __builtin_amdgcn_exp2f(mn == -__builtin_inff() ? s : s - mn);
        m = mn;
        l = l * alpha + p;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const float x = ld16<kBf16>(v[key * io.v_ts + 32 * n + 8 * (r >> 2) + 4 * h + (r & 3)]);
                const float pw = p != 0.f || s == -__builtin_inff() || __builtin_isfinite(x) ? p : 1.f;
                o[n][r] = __builtin_fmaf(pw, x, __builtin_isfinite(o[n][r]) ? o[n][r] * alpha : o[n][r]);
            }
    }
}

// kSplit: the work-group takes part blockIdx.y of its rows' keys (a kernel of its own: as one, whole calls take 3% longer).
template <int HD, bool kBf16, bool kCausal, bool kSplit>
__global__ __launch_bounds__(256, HD == 256 ? 1 : 2) void k_attn_varlen(const VarIo io) {
    typedef float f32x16 __attribute__((ext_vector_type(16)));
    using T = VarTile<HD>;
    using M = Mma<kBf16>;
    constexpr float kInf = __builtin_inff();
    constexpr int KB = T::kKeys, NB = KB / 32, KS = HD / 16, NT = HD / 32, CH = T::kChunks;
    const int tid = threadIdx.x, lane = tid & 63, c = lane & 31, h = lane >> 5;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    __shared__ __align__(16) unsigned char var_lds[var_lds_bytes<HD>()];
    // The tile of queries.  Tiles that see the most keys come first: with up to 64 sequences the tiles of all of them by
    // their place in the sequence, from the back, with more each sequence's own from the back.  Consecutive work-groups (of
    // different XCDs) take different KV heads, so that the query heads of one share its XCD's L2.
    const int item = (int)(blockIdx.x / io.nh), hh = blockIdx.x % io.nh, G = io.nh / io.nk, kvh = hh % io.nk;
    const int head = kvh * G + hh / io.nk;
    int q_first = 0, nq = 0, k_first = 0, nkeys = 0, t;
    if (io.n_seq <= 64) {
        if (lane < io.n_seq) {
            seq_rows(io.cu_q, io.Tq, lane, &q_first, &nq);
            seq_rows(io.cu_k, io.Tk, lane, &k_first, &nkeys);
        }
        const int tiles = nq > 0 ? (nq - 1) / kRows + 1 : 0;
        // tiles at place t of their sequence or behind it, over all sequences: the places from the back hold items 0, 1, ...
        auto from = [&](int place) { return wave_sum(max(tiles - place, 0)); };
        if (item >= from(0)) {
            if (kSplit && blockIdx.y == 0 && tid == 0) io.record[blockIdx.x].n = 0;
            return;
        }
        t = 0;                                   // the last place whose tiles end behind the item
        int step = 1;
        while (from(step) > item) step *= 2;
        for (step /= 2; step > 0; step /= 2)
            if (from(t + step) > item) t += step;
        uint64_t have = __builtin_amdgcn_ballot_w64(tiles > t);
        for (int skip = item - from(t + 1); skip > 0; --skip) have &= have - 1;
        const int b = __builtin_ctzll(have);
        q_first = __builtin_amdgcn_readlane(q_first, b);
        nq = __builtin_amdgcn_readlane(nq, b);
        k_first = __builtin_amdgcn_readlane(k_first, b);
        nkeys = __builtin_amdgcn_readlane(nkeys, b);
    } else {
        int64_t* const pre = reinterpret_cast<int64_t*>(var_lds);
        prefix_sums<256>(io.n_seq, pre, [&](int b) {
            int f, n;
            seq_rows(io.cu_q, io.Tq, b, &f, &n);
            return ((int64_t)n + kRows - 1) / kRows;
        });
        __syncthreads();
        const int at = (int)uniform(pre[io.n_seq]) - 1 - item;
        if (at < 0) {
            if (kSplit && blockIdx.y == 0 && tid == 0) io.record[blockIdx.x].n = 0;
            return;
        }
        const int b = find_item<256>(io.n_seq, pre, at);
        t = at - (int)uniform(pre[b]);
        seq_rows(io.cu_q, io.Tq, b, &q_first, &nq);
        seq_rows(io.cu_k, io.Tk, b, &k_first, &nkeys);
        q_first = __builtin_amdgcn_readfirstlane(q_first);
        nq = __builtin_amdgcn_readfirstlane(nq);
        k_first = __builtin_amdgcn_readfirstlane(k_first);
        nkeys = __builtin_amdgcn_readfirstlane(nkeys);
        __syncthreads();                         // (pre makes room for the first tile)
    }
    const int wg_q0 = t * kRows, q0 = wg_q0 + 32 * w;                    // first rows in the sequence
    const int past = nkeys - nq;                                         // row i attends keys 0 .. past + i
    const int wg_last = min(nq - wg_q0, kRows) - 1 + wg_q0;
    const int see = kCausal ? max(past + wg_last + 1, 0) : nkeys;        // keys of the work-group
    const int all_tiles = (int)(((int64_t)see + KB - 1) / KB);
    const int j0 = kSplit ? (int)((int64_t)all_tiles * blockIdx.y / io.splits) : 0;      // this part's tiles
    const int j1 = kSplit ? (int)((int64_t)all_tiles * (blockIdx.y + 1) / io.splits) : all_tiles;
    const int w_last = min(nq - q0, 32) - 1 + q0;                        // the wave's last row
    const int w_see = q0 >= nq ? 0 : kCausal ? past + w_last + 1 : nkeys;
    const int w_all = q0 >= nq ? 0 : kCausal ? past + q0 + 1 : nkeys;    // keys that all its rows see
    const bool row_ok = q0 + c < nq;
    const int lim = kCausal ? past + (row_ok ? q0 + c : nq - 1) : nkeys - 1;
    u32x4 qf[KS];
    {
        const uint16_t* qr = io.q + ((int64_t)q_first + (row_ok ? q0 + c : nq - 1)) * io.q_ts + head * io.q_hs + 8 * h;
#pragma unroll
        for (int st = 0; st < KS; ++st) qf[st] = *reinterpret_cast<const u32x4*>(qr + 16 * st);
    }
    const uint16_t* const kp = io.k + k_first * io.k_ts + kvh * io.k_hs;
    const uint16_t* const vp = io.v + k_first * io.v_ts + kvh * io.v_hs;
    // loads: a wave instruction fills 1 KB of LDS; instruction i of wave w holds rows (4 i + w) R .. (R = 512 / HD
    // rows), R rows apart by waves so that a lane's row keeps its low bits over i
    // (the whole offset goes into the load's vector offset: only that one is checked against the buffer's end)
    constexpr int R = 64 / CH, NI = T::kBytes / 4096;
    const int lrow = w * R + lane / CH, lpos = lane % CH;
    const int k_off = (int)(lrow * io.k_ts * 2) + 16 * (lpos ^ T::k_swz(lrow));
    const int v_off = (int)(lrow * io.v_ts * 2) + 16 * (lpos ^ T::v_swz(lrow));
    const int lds0 = __builtin_amdgcn_readfirstlane((int)(uintptr_t)(lds_u8*)var_lds);
    auto fetch = [&](int j, int buf) __attribute__((always_inline)) {
        const int k0 = j * KB;
        const int left = min(nkeys - k0, KB);
        const u32x4 kr = scalar_rsrc(kp + (int64_t)k0 * io.k_ts, (uint32_t)((left - 1) * (int)io.k_ts * 2 + HD * 2));
        const u32x4 vr = scalar_rsrc(vp + (int64_t)k0 * io.v_ts, (uint32_t)((left - 1) * (int)io.v_ts * 2 + HD * 2));
        const int dst = lds0 + buf * 2 * T::kBytes + w * 1024;
#pragma unroll
        for (int i = 0; i < NI; ++i) {
            load_lds(kr, dst + i * 4096, k_off + 8 * R * i * (int)io.k_ts);
            load_lds(vr, dst + T::kBytes + i * 4096, v_off + 8 * R * i * (int)io.v_ts);
        }
    };
    f32x16 o[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[n][r] = 0.f;
    // The weights enter the matrix cores in the type, as the values do (their sum stays in 32 bits): as two numbers each they
    // would double the products of V, half of what the matrix cores do here, for an output that is 2.1 to 2.5e-4 off
    // in fp16 where its own rounding is 1.8 to 2.0e-4 (bf16 2.1e-3 and 1.6e-3).
    // running maximum in powers of two, kept kUp below the largest score and raised when one exceeds it by more than kUp + 8:
    // probabilities stay at or below 2^15 in fp16, where many small ones (each over 2^-21 of the largest) keep their 11
    // bits, and at or below 2^8 in bf16, which holds small ones as well as large
    constexpr float kUp = kBf16 ? 0.f : 7.f;
    float m = -kInf, l = 0.f;
    // V^T reads: key and dimension that the lane names
    const int vi = lane & 15, vd = (lane >> 4 & 1) * 16 + 4 * (vi & 3), vk = 4 * h + (vi >> 2);
    auto tile = [&](int j, int buf, bool mask) __attribute__((always_inline)) {
        const unsigned char* kt = var_lds + buf * 2 * T::kBytes;
        const unsigned char* vt = kt + T::kBytes;
        f32x16 s[NB];
#pragma unroll
        for (int a = 0; a < NB; ++a) {
#pragma unroll
            for (int r = 0; r < 16; ++r) s[a][r] = 0.f;
            const int row = 32 * a + c;
#pragma unroll
            for (int st = 0; st < KS; ++st) {
                const u32x4 kf = *reinterpret_cast<const u32x4*>(kt + row * (HD * 2) + 16 * ((2 * st + h) ^ T::k_swz(row)));
                s[a] = M::mul(kf, qf[st], s[a]);
            }
        }
        if (mask) {
            asm volatile("");                    // (a branch: as selects these would run for every tile)
#pragma unroll
            for (int a = 0; a < NB; ++a)
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const int key = j * KB + 32 * a + 8 * (r >> 2) + 4 * h + (r & 3);
                    s[a][r] = key <= lim ? s[a][r] : -kInf;
                }
        }
        float mx = s[0][0];
#pragma unroll
        for (int a = 0; a < NB; ++a)
#pragma unroll
            for (int r = 0; r < 16; ++r) mx = fmaxf(mx, s[a][r]);
        mx = fmaxf(mx, __shfl_xor(mx, 32, 64)) * io.scale_log2;
        if (__builtin_amdgcn_ballot_w64(mx > m + (kUp + 8.f)) != 0) {
            const float mn = fmaxf(m, mx - kUp);
            const float alpha = m == mn ? 1.f : __builtin_amdgcn_exp2f(m - mn);
            m = mn;
            l *= alpha;
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int r = 0; r < 16; ++r) o[n][r] *= alpha;
        }
        const float nm = m == -kInf ? 0.f : -m;
#pragma unroll
        for (int a = 0; a < NB; ++a)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                s[a][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[a][r], io.scale_log2, nm));
                l += s[a][r];
            }
#pragma unroll
        for (int st = 0; st < KB / 16; ++st) {
            u32x4 pf;
#pragma unroll
            for (int e = 0; e < 4; ++e)
                pf[e] = pack16<kBf16>(s[st / 2][8 * (st & 1) + 2 * e], s[st / 2][8 * (st & 1) + 2 * e + 1]);
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                u32x4 vf;
#pragma unroll
                for (int a = 0; a < 2; ++a) {
                    const int row = 16 * st + 8 * a + vk, d = 32 * n + vd;
                    const u32x2 x = read_tr(vt + row * (HD * 2) + 16 * ((d / 8) ^ T::v_swz(row)) + 2 * (d % 8));
                    vf[2 * a] = x.x;
                    vf[2 * a + 1] = x.y;
                }
                o[n] = M::mul(vf, pf, o[n]);
            }
        }
    };
    if (j0 < j1) fetch(j0, 0);
    // the query is waited for here and not at its uses, where the wait would take in the next tile's loads
#pragma unroll
    for (int st = 0; st < KS; ++st) asm volatile("" : "+v"(qf[st]));
    for (int j = j0; j < j1; ++j) {
        const int buf = (j - j0) & 1;
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();                          // tile j is there, and nobody reads the other buffer any more
        if (j + 1 < j1) fetch(j + 1, buf ^ 1);
        const int k0 = j * KB;
        if (k0 < w_see) tile(j, buf, k0 + KB > w_all);
    }
    l += __shfl_xor(l, 32, 64);
    // A key that a row may not attend has probability zero there, and 0 * NaN or 0 * infinity must not reach the row:
    // where a sum is no finite number, the wave's rows are computed again by what they attend alone.
    float odd = 0.f;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int r = 0; r < 16; ++r) odd = __builtin_fmaf(0.f, o[n][r], odd);
    if (__builtin_amdgcn_ballot_w64(odd != 0.f) != 0)
        slow_rows<HD, kBf16>(io.q + ((int64_t)q_first + (row_ok ? q0 + c : nq - 1)) * io.q_ts + head * io.q_hs, kp, vp, io, j0 * KB,
                              min(w_see, j1 * KB), lim, h, o, m, l);
    if constexpr (kSplit) {
        const int64_t at = (int64_t)blockIdx.x * io.splits + blockIdx.y;
        if (blockIdx.y == 0 && tid == 0) io.record[blockIdx.x] = VarRecord{q_first, wg_q0, nq, head};
        if (!row_ok) return;
        float* const po = io.part_o + (at * kRows + 32 * w + c) * HD + 4 * h;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int g = 0; g < 4; ++g)
                *reinterpret_cast<f32x4*>(po + 32 * n + 8 * g) = f32x4{o[n][4 * g], o[n][4 * g + 1], o[n][4 * g + 2], o[n][4 * g + 3]};
        if (h == 0) {
            io.part_ml[(at * kRows + 32 * w + c) * 2] = m;
            io.part_ml[(at * kRows + 32 * w + c) * 2 + 1] = l;
        }
        return;
    }
    if (!row_ok) return;
    const float inv = l == 0.f ? 0.f : 1.f / l;
    uint16_t* const dst = io.out + ((int64_t)q_first + q0 + c) * io.o_ts + head * io.o_hs + 4 * h;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            uint32_t x[2];
#pragma unroll
            for (int e = 0; e < 2; ++e)
                x[e] = pack16<kBf16>(o[n][4 * g + 2 * e] * inv, o[n][4 * g + 2 * e + 1] * inv);
            *reinterpret_cast<u32x2*>(dst + 32 * n + 8 * g) = u32x2{x[0], x[1]};
        }
}

// The parts of 16 rows of an item, added up in their order: 16 threads a row.
template <int HD, bool kBf16>
__global__ __launch_bounds__(256) void k_varlen_combine(const VarIo io) {
    constexpr int N = HD / 16;
    const VarRecord rec = io.record[blockIdx.x];
    const int row = 16 * blockIdx.y + (threadIdx.x >> 4), d0 = (threadIdx.x & 15) * N;
    if (rec.n == 0 || rec.q0 + row >= rec.n) return;
    const int64_t base = (int64_t)blockIdx.x * io.splits * kRows + row;
    float m = -__builtin_inff(), l = 0.f;
    for (int i = 0; i < io.splits; ++i) m = fmaxf(m, io.part_ml[(base + (int64_t)i * kRows) * 2]);
    f32x4 acc[N / 4];
#pragma unroll
    for (int e = 0; e < N / 4; ++e) acc[e] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int i = 0; i < io.splits; ++i) {
        const int64_t at = base + (int64_t)i * kRows;
        const float pm = io.part_ml[at * 2], f = pm == m ? 1.f : __builtin_amdgcn_exp2f(pm - m);
        l = __builtin_fmaf(f, io.part_ml[at * 2 + 1], l);
#pragma unroll
        for (int e = 0; e < N / 4; ++e) {
            const f32x4 po = reinterpret_cast<const f32x4*>(io.part_o + at * HD + d0)[e];
#pragma unroll
            for (int i4 = 0; i4 < 4; ++i4)       // (0 * infinity: see slow_rows)
                acc[e][i4] = __builtin_fmaf(f != 0.f || __builtin_isfinite(po[i4]) ? f : 1.f, po[i4], acc[e][i4]);
        }
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    uint16_t* const dst = io.out + ((int64_t)rec.q_first + rec.q0 + row) * io.o_ts + rec.head * io.o_hs + d0;
#pragma unroll
    for (int e = 0; e < N / 4; ++e)
        reinterpret_cast<u32x2*>(dst)[e] = u32x2{pack16<kBf16>(acc[e][0] * inv, acc[e][1] * inv),
                                                 pack16<kBf16>(acc[e][2] * inv, acc[e][3] * inv)};
}

// Work-groups of a call at most (a tile of rows of a head each), and the parts that its keys are cut into: with few
// work-groups the keys of each are shared by up to 16, so that about 1024 run, each with at least 256 keys of a sequence of
// average length, or 1024 where there is a work-group for every CU already.  32 heads over 8, alone: 8 rows after 16000 keys
// 44 us and 8 sequences of such 233, where their bytes take 11 and 86.  With the reader of the cache before it: 8 rows
// after 16000 keys 298 -> 60 us, 128 rows after 4000 92 -> 40; 8 sequences of 8 rows after 16000 keys 440 -> 380; 1024 rows
// after 500 keys in three parts of 500 42 -> 51, so they stay whole.
int64_t var_items(int64_t n_seq, int64_t Tq, int64_t nh) { return ((Tq + kRows - 1) / kRows + (n_seq < Tq ? n_seq : Tq)) * nh; }
int var_splits(int64_t n_seq, int64_t Tk, int64_t items) {
    const int64_t a = items > 0 ? 1024 / items : 1, b = Tk / (n_seq * (items < 256 ? 256 : 1024)), c = a < b ? a : b;
    return (int)(c < 2 ? 1 : c > 16 ? 16 : c);
}
int64_t var_ws(int64_t items, int splits, int64_t hd) {
    return splits > 1 ? items * (splits * (int64_t)kRows * (hd + 2) * 4 + (int64_t)sizeof(VarRecord)) : 0;
}

template <int HD>
void launch(const VarIo& io, int dtype, int causal, unsigned grid, hipStream_t st) {
    const dim3 g(grid, (unsigned)io.splits), c(grid, kRows / 16);
    auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, g, dim3(256), 0, st, io); };
    if (io.splits == 1) {
        if (dtype && causal) go(k_attn_varlen<HD, true, true, false>);
        else if (dtype) go(k_attn_varlen<HD, true, false, false>);
        else if (causal) go(k_attn_varlen<HD, false, true, false>);
        else go(k_attn_varlen<HD, false, false, false>);
        return;
    }
    if (dtype && causal) go(k_attn_varlen<HD, true, true, true>);
    else if (dtype) go(k_attn_varlen<HD, true, false, true>);
    else if (causal) go(k_attn_varlen<HD, false, true, true>);
    else go(k_attn_varlen<HD, false, false, true>);
    if (dtype) hipLaunchKernelGGL((k_varlen_combine<HD, true>), c, dim3(256), 0, st, io);
    else hipLaunchKernelGGL((k_varlen_combine<HD, false>), c, dim3(256), 0, st, io);
}

}  // namespace
}  // namespace sx8

extern "C" int64_t sx8_attn_varlen_workspace_bytes(int64_t n_seq, int64_t Tq, int64_t Tk, int32_t nh, int32_t hd) {
    using namespace sx8;
    if (n_seq <= 0 || n_seq > kKv4MaxSlots || Tq < 0 || Tk < 0 || nh <= 0) return -1;
    const int64_t items = var_items(n_seq, Tq, nh);
    return var_ws(items, var_splits(n_seq, Tk, items), hd);
}

extern "C" int32_t sx8_attn_varlen(const void* q, const void* k, const void* v, void* out, const int32_t* cu_q,
                                   const int32_t* cu_k, int64_t n_seq, int64_t Tq, int64_t Tk, int32_t nh, int32_t nk,
                                   int32_t hd, int64_t q_ts, int64_t q_hs, int64_t k_ts, int64_t k_hs, int64_t v_ts,
                                   int64_t v_hs, int64_t o_ts, int64_t o_hs, float scale, int32_t causal, int32_t dtype,
                                   void* workspace, int64_t workspace_bytes, void* stream) {
    using namespace sx8;
    const char* what = "sx8_attn_varlen";
    if (!cu_q || !cu_k || (Tq > 0 && (!q || !out)) || (Tk > 0 && (!k || !v)))
        return fail(SX8_ERR_INVALID, "%s: null pointer", what);
    if ((hd != 64 && hd != 128 && hd != 256) || nk <= 0 || nh <= 0 || nh % nk || nh > 65536)
        return fail(SX8_ERR_INVALID, "%s: bad shape (hd 64, 128 or 256, nh a multiple of nk)", what);
    if (n_seq <= 0 || n_seq > kKv4MaxSlots || Tq < 0 || Tq > 0x7FFFFF00 || Tk < 0 || Tk > 0x7FFFFF00)
        return fail(SX8_ERR_INVALID, "%s: bad sizes (n_seq 1..%d, Tq and Tk below 2^31 - 256)", what, kKv4MaxSlots);
    if (dtype != 0 && dtype != 1) return fail(SX8_ERR_INVALID, "%s: dtype must be 0 (fp16) or 1 (bf16)", what);
    if (!(scale > 0.f) || !(scale < __builtin_inff()))
        return fail(SX8_ERR_INVALID, "%s: scale must be positive and finite", what);
    if (!aligned(q, 16) || !aligned(k, 16) || !aligned(v, 16) || !aligned(out, 16) || !aligned(cu_q, 4) || !aligned(cu_k, 4))
        return fail(SX8_ERR_INVALID, "%s: q, k, v and out must be 16-byte aligned, cu_q and cu_k 4-byte", what);
    const int64_t strides[8] = {q_ts, q_hs, k_ts, k_hs, v_ts, v_hs, o_ts, o_hs};
    for (int i = 0; i < 8; ++i)
        if (strides[i] % 8 || strides[i] < 0 || strides[i] > (int64_t)1 << 40)
            return fail(SX8_ERR_INVALID, "%s: strides must be multiples of 8", what);
    if (Tq > 0 && !rows_apart(o_ts, o_hs, Tq, nh, hd)) return fail(SX8_ERR_INVALID, "%s: rows of out overlap", what);
    if (k_ts < hd || v_ts < hd || k_ts > 1 << 23 || v_ts > 1 << 23)     // (a tile's rows lie within 32-bit offsets)
        return fail(SX8_ERR_INVALID, "%s: the token strides of k and v must be hd .. 2^23", what);
    const int64_t items = var_items(n_seq, Tq, nh);
    if (items > 0x7FFFFFFF) return fail(SX8_ERR_UNSUPPORTED, "%s: over 2^31 tiles of rows", what);
    int splits = var_splits(n_seq, Tk, items);
    if (splits > 1 && !workspace) splits = 1;
    if (splits > 1 && (workspace_bytes < var_ws(items, splits, hd) || !aligned(workspace, 256)))
        return fail(SX8_ERR_INVALID, "%s: workspace needs %lld bytes, 256-byte aligned", what,
                    (long long)var_ws(items, splits, hd));
    if (Tq == 0) return ok();
    VarIo io{(const uint16_t*)q, (const uint16_t*)k, (const uint16_t*)v, (uint16_t*)out, cu_q, cu_k, q_ts, q_hs, k_ts,
             k_hs, v_ts, v_hs, o_ts, o_hs, (int)Tq, (int)Tk, (int)n_seq, nh, nk, scale * 1.4426950408889634f, splits,
             nullptr, nullptr, nullptr};
    if (splits > 1) {
        io.record = reinterpret_cast<VarRecord*>(workspace);
        io.part_o = reinterpret_cast<float*>(io.record + items);
        io.part_ml = io.part_o + items * splits * kRows * (int64_t)hd;
    }
    const hipStream_t st = as_stream(stream);
    if (hd == 64) launch<64>(io, dtype, causal, (unsigned)items, st);
    else if (hd == 128) launch<128>(io, dtype, causal, (unsigned)items, st);
    else launch<256>(io, dtype, causal, (unsigned)items, st);
    return check_launch(what);
}
