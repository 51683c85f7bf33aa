// sx8_draft.hip -- drafted tokens: masks of their trees, and verification against the target (include/sx8_draft.h).
#include "sx8_draft.h"

#include <type_traits>

#include "sx8_host.h"
#include "sx8_kv4_dev.h"

namespace sx8 {
namespace {

constexpr int kMaxWords = 4;

// ---- trees -------------------------------------------------------------------------------------
// A work-group takes a slot.  Ancestors by doubling: after round i a row knows those up to 2^i steps above it and the
// row that many steps up, so that a chain of 256 takes 8 rounds.
__global__ __launch_bounds__(256) void k_draft_tree(const int32_t* parents, const int32_t* cu, Kv4Shape sh, int words,
                                                    uint64_t* mask, int32_t* depth) {
    __shared__ uint64_t m[64 * kMaxWords][kMaxWords];
    __shared__ int up[64 * kMaxWords], d[64 * kMaxWords];
    int first, n;
    kv4_rows(sh, cu, blockIdx.x, &first, &n);
    const int i = threadIdx.x, most = min(n, 64 * words);
    int at = -1;
    if (i < most) {
        at = parents[first + i];
        if (at < 0 || at >= i) at = -1;
        for (int w = 0; w < words; ++w) m[i][w] = w == i / 64 ? 1ull << i % 64 : 0;
        d[i] = at >= 0;
        up[i] = at;
    }
    while (__syncthreads_or(at >= 0)) {
        uint64_t more[kMaxWords];
        int next = -1, steps = 0;
        if (at >= 0) {
            for (int w = 0; w < words; ++w) more[w] = m[at][w];
            next = up[at];
            steps = d[at];
        }
        __syncthreads();
        if (at >= 0) {
            for (int w = 0; w < words; ++w) m[i][w] |= more[w];
            d[i] += steps;
            up[i] = at = next;
        }
    }
    for (int r = i; r < n; r += 256) {
        for (int w = 0; w < words; ++w) mask[((int64_t)first + r) * words + w] = r < most ? m[r][w] : 0;
        depth[first + r] = r < most ? d[r] : -(1 << 30);
    }
}

// ---- verification ------------------------------------------------------------------------------
// Two launches: every row's largest logit and the sum of its weights exp((logit - largest) / temperature), by
// parts of kPart logits; then a work-group for each slot walks its tree, where a test needs one logit of a row, and draws the
// next token, where the parts' sums say in which part it lies.  With draft probabilities a refused token costs a sum over the
// vocabulary: the walk stops there, a launch sums the parts of all slots that wait, and a second walk goes on (further
// refusals, which trees can have, it sums by itself).  All in binary64: the token must not depend on the order in which 150000
// weights were added, and of so many borders of the cumulated sum one lies within a binary32 rounding of u once in some
// hundred draws.  The first launch reads all rows, though a walk needs only those that it comes to (of the 515 rows below 20 to
// 24, of the 187 56 to 70): no work-group waits for another then, and a row at a time is what a walk would take otherwise.
// The rows of 16 trees (515 of 151936 float32 logits, 313 MB) take 62 us, where reading them takes 49 (18 instructions a logit, nine of
// them of 64 bits), the walk 16; 32 chains of 187 rows with draft probabilities 29, 8.2, 14.6 (the left sums) and 10; a chain of
// five whose first token is refused 5 and 10.8, which are about seven dependent round trips.
constexpr int kPart = 4096, kRowThreads = 256, kWalkThreads = 1024, kNear = 256;

struct RowPart {
    double sum;                           // of exp((x - top) / temperature), or 0 (greedy)
    float top;                            // largest logit of the part (-infinity: none)
    int32_t arg;                          // its first index
};
static_assert(sizeof(RowPart) == 16, "part");

// Where a walk waits for the sums of its slot's parts: weights max(a w / sum - b q, 0) of row `cur`, for the child `row`.
struct Wait {
    double a, b;
    int32_t cur, count, row, open;        // open 0: the slot is done
};

struct VerifyIo {
    const void* logits;
    int64_t stride;
    const int64_t* tokens;
    const int32_t *parents, *cu;
    Kv4Shape sh;
    int64_t V;
    int parts;                            // of a row
    const float *u, *temperature;
    float t;
    const int32_t* depth;                 // below zero: the row is no part of its tree (null: all are)
    const void* probs;
    int64_t probs_stride;
    int32_t *path, *counts;
    int64_t* next;
    RowPart* part;                        // [rows][parts]
    RowPart* row;                         // [rows]: the whole row
    double* p;                            // [rows]: probability of a row's token at its parent, below zero: none
    int32_t* gone;                        // [rows]: rows of a slot whose tokens are out of p at its current row
    double* slot_sum;                     // [n_slots][parts]: sums of what is left of p
    Wait* wait;                           // [n_slots]
};

template <int kType>                      // 0 fp16, 1 bf16, 2 float32
__device__ __forceinline__ float value(const void* base, int64_t at) {
    if constexpr (kType == 2) return static_cast<const float*>(base)[at];
    else return ld16<kType == 1>(static_cast<const uint16_t*>(base)[at]);
}
__device__ __forceinline__ float logit(float x) { return x == x ? x : -__builtin_inff(); }

// exp((x - top) / temperature) for x <= top; scale = log2(e) / temperature.  2^y = 2^n 2^f with n the nearest integer, 2^f by its
// interpolation in the Chebyshev nodes of [-1/2, 1/2] (degree 10: within 3e-16 of itself).  An infinite top has the weights
// of a row of -infinity and 0.
struct Weigh {
    double top, scale;
    bool all;                             // top is infinite
    __device__ __forceinline__ Weigh(float t, double s) : top(t == __builtin_inff() ? 0.0 : t), scale(s), all(t == __builtin_inff()) {}
    __device__ __forceinline__ double operator()(float x) const {
        if (all) return x == __builtin_inff() ? 1.0 : 0.0;
        double y = ((double)x - top) * scale;
        const bool none = !(y >= -1000.0);                           // (-infinity, and 0 * infinity)
        y = none ? 0.0 : y;
        const double shifted = y + 0x1.8p52, f = y - (shifted - 0x1.8p52);
        double r = 0x1.e6063f7217bc6p-28;
        r = __builtin_fma(r, f, 0x1.b675bca4eeebbp-24);
        r = __builtin_fma(r, f, 0x1.62bfd47773353p-20);
        r = __builtin_fma(r, f, 0x1.ffcb54062e698p-17);
        r = __builtin_fma(r, f, 0x1.430913096fd9fp-13);
        r = __builtin_fma(r, f, 0x1.5d87fe9d7a584p-10);
        r = __builtin_fma(r, f, 0x1.3b2ab6fba1ddap-7);
        r = __builtin_fma(r, f, 0x1.c6b08d703ce49p-5);
        r = __builtin_fma(r, f, 0x1.ebfbdff82c598p-3);
        r = __builtin_fma(r, f, 0x1.62e42fefa3a19p-1);
        r = __builtin_fma(r, f, 1.0);
        const uint64_t bits = __builtin_bit_cast(uint64_t, r) + (__builtin_bit_cast(uint64_t, shifted) << 52);
        return none ? 0.0 : __builtin_bit_cast(double, bits);
    }
};
__device__ __forceinline__ float temperature_of(const VerifyIo& io, int slot) { return io.temperature ? io.temperature[slot] : io.t; }
__device__ __forceinline__ double scale_of(float temperature) { return 1.4426950408889634 / (double)temperature; }

__device__ __forceinline__ double lane_of_double(double v, int lane) {
    return __builtin_bit_cast(double, lane_of(__builtin_bit_cast(int64_t, v), lane));
}
__device__ __forceinline__ double wave_add(double v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}
// The sum over the lanes up to this one.
__device__ __forceinline__ double wave_prefix_sum(double v) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const double u = __shfl_up(v, o, 64);
        if (lane >= o) v += u;
    }
    return v;
}
// The sum over the work-group's kT threads, the same in every thread.
template <int kT>
__device__ __forceinline__ double group_add(double v) {
    __shared__ double s[kT / 64];
    v = wave_add(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = v;
    __syncthreads();
    double r = 0.0;
#pragma unroll
    for (int i = 0; i < kT / 64; ++i) r += s[i];
    return r;
}
// (top, first index) of two candidates
__device__ __forceinline__ void better(float& top, int& arg, float t, int a) {
    if (t > top || (t == top && a < arg)) {
        top = t;
        arg = a;
    }
}

// The slot that has row r, or -1.  mine: where slot `lane` ends, 2^31 - 1 for none; begin: where slot 0 begins.
__device__ __forceinline__ int slot_of(const Kv4Shape& sh, const int32_t* cu, int r, int mine, int begin) {
    const int lane = threadIdx.x & 63;
    // (ends grow: the slots that end at or before r come first; 64 at a time)
    int s = __builtin_popcountll(__builtin_amdgcn_ballot_w64(mine <= r));
    if (s < 64) {
        if (s > 0) begin = __builtin_amdgcn_readlane(mine, s - 1);
    } else {
        for (int k = 64; k == 64 && s < sh.n_slots; s += k) {
            const int at = s + lane;
            k = __builtin_popcountll(__builtin_amdgcn_ballot_w64(at < sh.n_slots && cu[at + 1] <= r));
        }
        if (s < sh.n_slots) begin = cu[s];
    }
    return s >= sh.n_slots || begin > r ? -1 : s;
}

// kWide: rows begin on 16 bytes, and a thread takes 16 bytes at a time.
template <int kType, bool kWide>
__global__ __launch_bounds__(kRowThreads) void k_verify_rows(const VerifyIo io) {
    constexpr int kE = kPart / kRowThreads, kN = !kWide ? 1 : kType == 2 ? 4 : 8;
    const int r = blockIdx.x, part = blockIdx.y, tid = threadIdx.x, lane = tid & 63;
    const int64_t base = (int64_t)part * kPart, from = r * io.stride + base;
    const int n = (int)min((int64_t)kPart, io.V - base);
    const int mine = lane < io.sh.n_slots ? io.cu[lane + 1] : 0x7FFFFFFF, begin = io.cu[0];   // (asked for before the logits)
    float x[kE], top = -__builtin_inff();
    auto place = [&](int i) { return (i / kN * kRowThreads + tid) * kN + i % kN; };
    if constexpr (kWide) {
        u32x4 raw[kE / kN];
        auto load = [&](int at) { return *reinterpret_cast<const u32x4*>(static_cast<const char*>(io.logits) + (from + at) * (kType == 2 ? 4 : 2)); };
        if (n == kPart) {
#pragma unroll
            for (int i = 0; i < kE / kN; ++i) raw[i] = load(place(i * kN));
        } else {
#pragma unroll
            for (int i = 0; i < kE / kN; ++i) {
                constexpr uint32_t kNone = kType == 2 ? 0xFF800000u : kType == 1 ? 0xFF80FF80u : 0xFC00FC00u;   // -infinity
                raw[i] = u32x4{kNone, kNone, kNone, kNone};
                const int at = place(i * kN);
                if (at + kN <= n) raw[i] = load(at);
                else
                    for (int e = 0; e < kN && at + e < n; ++e) {
                        if constexpr (kType == 2) raw[i][e] = __builtin_bit_cast(uint32_t, value<2>(io.logits, from + at + e));
                        else raw[i][e >> 1] = (raw[i][e >> 1] & (e & 1 ? 0xFFFFu : 0xFFFF0000u)) | (uint32_t)static_cast<const uint16_t*>(io.logits)[from + at + e] << 16 * (e & 1);
                    }
            }
        }
#pragma unroll
        for (int i = 0; i < kE; ++i) {
            if constexpr (kType == 2) x[i] = __builtin_bit_cast(float, (uint32_t)raw[i / kN][i % kN]);
            else x[i] = ld16<kType == 1>(half_of(raw[i / kN][i % kN >> 1], i));
        }
    } else {
#pragma unroll
        for (int i = 0; i < kE; ++i) x[i] = place(i) < n ? value<kType>(io.logits, from + place(i)) : -__builtin_inff();
    }
    // (a NaN is no maximum here, equals none, and weighs what -infinity does: fmaxf takes the other number)
    const int slot = slot_of(io.sh, io.cu, r, mine, begin);
    if (slot < 0) return;
    const float temp = temperature_of(io, slot);
#pragma unroll
    for (int i = 0; i < kE; ++i) top = fmaxf(top, x[i]);
    float all = top;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) all = fmaxf(all, __shfl_xor(all, o, 64));
    __shared__ float tops[kRowThreads / 64];
    __shared__ double root[32];
    __shared__ int first;
    if (tid < 32) root[tid] = Weigh(0.f, 1.0 / 32.0)(tid - 32) * 2.0;
    if (lane == 0) tops[tid >> 6] = all;
    if (tid == 0) first = 0x7FFFFFFF;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kRowThreads / 64; ++i) all = fmaxf(all, tops[i]);
    if (all > -__builtin_inff() && top == all) {
        int arg = 0x7FFFFFFF;
#pragma unroll
        for (int i = kE - 1; i >= 0; --i)
            if (x[i] == all) arg = place(i);
        atomicMin(&first, arg);
    }
    double sum = 0.0;
    if (temp > 0.f && all > -__builtin_inff()) {
        // 2^y as 2^(j / 32) from LDS times 2^f by its interpolation in the Chebyshev nodes of [-1/64, 1/64] (degree 4, within
        // 8e-14 of itself), where no weight is below e^-690 for it: 9 operations of 64 bits a logit, 18 by Weigh.  32 y is
        // x scale - top32 for an integer top32, and the sum takes the rest of the top once.
        // (a temperature that the logits' float32 steps do not resolve leaves no such clamp)
        const float lowest = all - 680.f * temp;
        const double gap = (double)all - (double)lowest, scale = 32.0 * scale_of(temp), top32 = rint((double)all * scale);
        if (all < __builtin_inff() && lowest > -__builtin_inff() && gap >= 600.0 * (double)temp && gap <= 690.0 * (double)temp &&
            __builtin_fabs(top32) < 0x1p40) {
            auto root_of = [](double f) {                            // 2^(f / 32)
                double r = __builtin_fma(0x1.3b2b1bee88b09p-27, f, 0x1.c6b167e571135p-20);
                r = __builtin_fma(r, f, 0x1.ebfbdff8131c3p-13);
                r = __builtin_fma(r, f, 0x1.62e42fef6d01ap-6);
                return __builtin_fma(r, f, 1.0);
            };
            const double c = 0x1.8p52 - top32;
#pragma unroll
            for (int i = 0; i < kE; ++i) {
                const double v = fmaxf(x[i], lowest), shifted = __builtin_fma(v, scale, c), f = __builtin_fma(v, scale, c - shifted);
                const int n = (int)__builtin_bit_cast(uint64_t, shifted);
                const uint64_t bits = __builtin_bit_cast(uint64_t, root[n & 31]) + ((uint64_t)(uint32_t)(n >> 5) << 52);
                sum = __builtin_fma(__builtin_bit_cast(double, bits), root_of(f), sum);
            }
            sum *= root_of(__builtin_fma(-(double)all, scale, top32));
        } else {
            const Weigh w(all, scale_of(temp));
#pragma unroll 1
            for (int i = 0; i < kE; ++i) {
                float v = x[0];
#pragma unroll
                for (int j = 1; j < kE; ++j) v = i == j ? x[j] : v;
                sum += w(v);
            }
        }
    }
    sum = group_add<kRowThreads>(sum);                               // (behind its barriers `first` is whole)
    if (tid == 0) io.part[(int64_t)r * io.parts + part] = RowPart{sum, all, all > -__builtin_inff() ? (int)base + first : 0x7FFFFFFF};
}

// A row's parts as one (wave-wide; every lane gets it).
__device__ __forceinline__ RowPart whole_row(const VerifyIo& io, int64_t row, bool greedy, double scale) {
    const int lane = threadIdx.x & 63;
    const RowPart* const p = io.part + row * io.parts;
    RowPart r = {0.0, -__builtin_inff(), 0x7FFFFFFF};
    for (int i = lane; i < io.parts; i += 64) better(r.top, r.arg, p[i].top, p[i].arg);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) better(r.top, r.arg, __shfl_xor(r.top, o, 64), __shfl_xor(r.arg, o, 64));
    if (greedy) return r;
    const Weigh w(r.top, scale);
    for (int i = lane; i < io.parts; i += 64)
        if (p[i].top > -__builtin_inff()) r.sum += p[i].sum * w(p[i].top);
    r.sum = wave_add(r.sum);
    return r;
}

// The sums of the parts of rows that wait: work-group (part, slot).
template <int kType, int kProbs>
__global__ __launch_bounds__(kRowThreads) void k_verify_left(const VerifyIo io) {
    const int slot = blockIdx.y, part = blockIdx.x, tid = threadIdx.x;
    const Wait wt = io.wait[slot];
    if (!wt.open) return;
    int first, n;
    kv4_rows(io.sh, io.cu, slot, &first, &n);
    const int64_t row = (int64_t)first + wt.cur, base = (int64_t)part * kPart;
    const RowPart rs = io.row[row];
    const Weigh w(rs.top, scale_of(temperature_of(io, slot)));
    const double a = wt.a / rs.sum;
    const int m = (int)min((int64_t)kPart, io.V - base);
    double s = 0.0;
    for (int e0 = 0; e0 < m; e0 += 8 * kRowThreads) {
        float x[8], q[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int e = e0 + i * kRowThreads + tid;
            x[i] = e < m ? value<kType>(io.logits, row * io.stride + base + e) : -__builtin_inff();
            q[i] = e < m ? value<kProbs>(io.probs, row * io.probs_stride + base + e) : 0.f;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) s += fmax(a * w(logit(x[i])) - wt.b * (double)q[i], 0.0);
    }
    s = group_add<kRowThreads>(s);
    if (tid == 0) io.slot_sum[(int64_t)slot * io.parts + part] = s;
}

// kProbs -1: no draft probabilities.  kGoOn: the second walk, from where the first one waits.
template <int kType, int kProbs, bool kGoOn>
__global__ __launch_bounds__(kWalkThreads) void k_verify_walk(const VerifyIo io) {
    constexpr bool kFirst = kProbs >= 0 && !kGoOn;                    // (stops at a refused token)
    const int slot = blockIdx.x, tid = threadIdx.x, lane = tid & 63;
    const float temp = temperature_of(io, slot);                     // (asked for with cu)
    int first, n;
    kv4_rows(io.sh, io.cu, slot, &first, &n);
    // a slot without rows, or whose first one is no part of a tree
    auto none = [&]() {
        for (int i = tid; i < n; i += kWalkThreads) io.path[first + i] = -1;
        if (tid == 0) {
            io.counts[slot] = 0;
            io.next[slot] = -1;
            if constexpr (kProbs >= 0) io.wait[slot].open = 0;
        }
    };
    if (n == 0) return none();
    const int root = io.depth ? io.depth[first] : 0;
    // parent, token and uniform of row i0 + lane, the first ones on their way before the sums of rows
    int par = -1;
    int64_t tok = -1;
    float un = 0.f;
    auto load_rows = [&](int i0) {
        const int row = i0 + lane;
        par = row > 0 && row < n ? io.parents[first + row] : -1;
        tok = row < n ? io.tokens[first + row] : -1;
        un = row < n && io.u ? io.u[first + row] : 0.f;
    };
    if constexpr (!kGoOn) load_rows(0);
    const float u0 = io.u ? io.u[first] : 0.f;
    if (root < 0) return none();
    const bool greedy = !(temp > 0.f);
    const double scale = greedy ? 0.0 : scale_of(temp);
    // the slot's lists: in LDS where they fit and nobody else reads them
    __shared__ RowPart row_lds[kProbs < 0 ? kNear : 1];
    __shared__ double p_lds[kProbs < 0 ? kNear : 1], sum_lds[kNear];
    __shared__ int gone_lds[kNear];
    const bool near = kProbs < 0 && n <= kNear;
    RowPart* const whole = near ? row_lds : io.row + first;
    double* const prob = near ? p_lds : io.p + first;
    double* const slot_sum = !kGoOn && io.parts <= kNear ? sum_lds : io.slot_sum + (int64_t)slot * io.parts;
    int* const gone = n <= kNear ? gone_lds : io.gone + first;       // rows of the tokens that are out of p
    int cur = 0, count = 1, n_gone = 0, i0 = 0;
    double left = 1.0, a = 1.0, b = 0.0, total = 1.0;
    uint64_t above = ~0ull;                                           // rows of the first 64 that are still to be tried
    if constexpr (kGoOn) {
        const Wait wt = io.wait[slot];
        if (!wt.open) return;
        cur = wt.cur;
        count = wt.count;
        i0 = wt.row & ~63;
        load_rows(i0);
        above = wt.row % 64 == 63 ? 0ull : ~0ull << (wt.row % 64 + 1);
        a = wt.a;
        b = wt.b;
        double s = 0.0;
        for (int i = tid; i < io.parts; i += kWalkThreads) s += slot_sum[i];
        total = group_add<kWalkThreads>(s);
        if (!(total > 0.0)) {
            a = total = 1.0;
            b = 0.0;
        }
    } else {
        // whole rows, then every token's probability at its parent: all of them at once
        for (int i = tid >> 6; i < n; i += kWalkThreads / 64) {
            const RowPart r = whole_row(io, (int64_t)first + i, greedy, scale);
            if (lane == 0) whole[i] = r;
        }
        for (int i = tid; i < n; i += kWalkThreads) io.path[first + i] = i == 0 ? 0 : -1;
        __syncthreads();
        for (int i = tid; i < n; i += kWalkThreads) {
            const int up = i < 64 ? par : io.parents[first + i];
            const int64_t x = i < 64 ? tok : io.tokens[first + i];
            const int deep = io.depth ? io.depth[first + i] : 0;
            double p = -1.0;
            if (i > 0 && deep >= 0 && up >= 0 && up < i && x >= 0 && x < io.V) {
                const RowPart r = whole[up];
                if (r.top > -__builtin_inff()) {
                    if (greedy) p = x == r.arg;
                    else p = Weigh(r.top, scale)(logit(value<kType>(io.logits, ((int64_t)first + up) * io.stride + x))) / r.sum;
                }
            }
            prob[i] = p;
        }
        __syncthreads();
    }
    RowPart rs = whole[cur];
    // the weight that is left of token x at the current row
    auto weigh = [&](const Weigh& w, double per, int64_t x, double cb) -> double {
        double v = w(logit(value<kType>(io.logits, ((int64_t)first + cur) * io.stride + x))) * per;
        if constexpr (kProbs >= 0) {
            if (cb != 0.0) v = fmax(v - cb * (double)value<kProbs < 0 ? 0 : kProbs>(io.probs, ((int64_t)first + cur) * io.probs_stride + x), 0.0);
        }
        return v;
    };
    auto token_of = [&](int row) { return io.tokens[first + row]; };
    // (a cu that runs backwards gives slots the same rows, and their lists in memory the same places)
    auto gone_row = [&](int i) { return (int)min((unsigned)gone[i], (unsigned)n - 1u); };
    auto is_gone = [&](int64_t x) {
        for (int i = 0; i < n_gone; ++i)
            if (token_of(gone_row(i)) == x) return true;
        return false;
    };
    // the sums of the parts for coefficients a, b by this work-group; their sum
    auto sum_parts = [&]() {
        const Weigh w(rs.top, scale);
        const double per = a / rs.sum;
        double all = 0.0;
        for (int part = 0; part < io.parts; ++part) {
            double s = 0.0;
            const int64_t base = (int64_t)part * kPart, m = min((int64_t)kPart, io.V - base);
            for (int e = tid; e < m; e += kWalkThreads) s += weigh(w, per, base + e, b);
            s = group_add<kWalkThreads>(s);
            if (tid == 0) slot_sum[part] = s;
            all += s;
        }
        return all;
    };
    // the walk: every wave does it alike, a row a lane
    for (bool loaded = true; i0 < n; i0 += 64, above = ~0ull, loaded = false) {
        if (!loaded) load_rows(i0);
        const double pr = i0 + lane < n ? prob[i0 + lane] : -1.0;
        double qr = 0.0;
        if constexpr (kProbs >= 0)
            if (pr >= 0.0 && !greedy) qr = (double)value<kProbs < 0 ? 0 : kProbs>(io.probs, ((int64_t)first + par) * io.probs_stride + tok);
        uint64_t todo = __builtin_amdgcn_ballot_w64(par == cur && pr >= 0.0) & above;
        while (todo) {
            const int k = __builtin_ctzll(todo);
            todo &= todo - 1;
            const double p = lane_of_double(pr, k), uk = lane_of_double((double)un, k);
            bool keep;
            if (greedy) {
                keep = p > 0.0;
            } else if constexpr (kProbs < 0) {
                const int64_t x = lane_of(tok, k);
                const bool some = p > 0.0 && !is_gone(x);
                keep = some && uk < 1.0 && uk * left < p;
                if (some && !keep) {
                    __syncthreads();
                    if (tid == 0) gone[n_gone] = i0 + k;
                    __syncthreads();
                    ++n_gone;
                    left -= p;
                }
            } else {
                const double q = lane_of_double(qr, k), now = (b != 0.0 ? fmax(a * p - b * q, 0.0) : p) / total;
                keep = now > 0.0 && uk * q < now;
                if (!keep) {
                    // max(p - q, 0) with p = max(a w - b q, 0) / total: coefficients a / total and b / total + 1
                    a /= total;
                    b = b / total + 1.0;
                    if constexpr (kFirst) {
                        if (tid == 0) io.wait[slot] = Wait{a, b, cur, count, i0 + k, 1};
                        return;
                    }
                    total = sum_parts();
                    if (!(total > 0.0)) {
                        a = total = 1.0;
                        b = 0.0;
                    }
                }
            }
            if (keep) {
                cur = i0 + k;
                rs = whole[cur];
                if (tid == 0) io.path[first + count] = cur;
                ++count;
                n_gone = 0;
                left = a = total = 1.0;
                b = 0.0;
                todo = __builtin_amdgcn_ballot_w64(par == cur && pr >= 0.0 && lane > k);
            }
        }
    }
    if (tid == 0) {
        io.counts[slot] = count;
        if constexpr (kProbs >= 0) io.wait[slot].open = 0;
    }
    if (greedy || !(rs.top > -__builtin_inff())) {
        if (tid == 0) io.next[slot] = rs.top > -__builtin_inff() ? rs.arg : -1;
        return;
    }
    // the sums of the parts of what is left
    const Weigh w(rs.top, scale);
    const double per = a / rs.sum;
    if (b == 0.0) {
        // A part's sum without the tokens that are out: less their weights, which keeps the sums' precision where most of the
        // part is left; summed anew where less than 2^-20 of it is.
        const RowPart* const rp = io.part + ((int64_t)first + cur) * io.parts;
        auto fill = [&]() {
            __syncthreads();
            double s = 0.0;
            bool anew = false;
            for (int i = tid; i < io.parts; i += kWalkThreads) {
                const double of = rp[i].top > -__builtin_inff() ? rp[i].sum * w(rp[i].top) / rs.sum : 0.0;
                double v = of;
                for (int j = 0; j < n_gone; ++j)
                    if (token_of(gone_row(j)) / kPart == i) v -= prob[gone_row(j)];
                const bool again = v < of * 0x1p-20;
                anew |= again;
                slot_sum[i] = again ? -1.0 : v;
                s += again ? 0.0 : v;
            }
            if (__syncthreads_or(anew))
                for (int part = 0; part < io.parts; ++part) {
                    if (slot_sum[part] >= 0.0) continue;             // (alike in all threads)
                    const int64_t base = (int64_t)part * kPart, m = min((int64_t)kPart, io.V - base);
                    double v = 0.0;
                    for (int e = tid; e < m; e += kWalkThreads) v += is_gone(base + e) ? 0.0 : weigh(w, per, base + e, 0.0);
                    v = group_add<kWalkThreads>(v);
                    if (tid == 0) {
                        slot_sum[part] = v;
                        s += v;
                    }
                    __syncthreads();
                }
            return group_add<kWalkThreads>(s);
        };
        total = fill();
        if (!(total > 0.0)) {                 // nothing left: the target's own
            n_gone = 0;
            total = fill();
        }
    }
    __syncthreads();
    // the part in which the sum passes u * total (or, by roundings, the last one that has any)
    const double goal = (double)u0 * total;
    double before = 0.0, last_before = 0.0;
    int part = -1, last = 0;
    for (int p0 = 0; p0 < io.parts && part < 0; p0 += 64) {
        const double s = p0 + lane < io.parts ? slot_sum[p0 + lane] : 0.0, end = wave_prefix_sum(s);
        const uint64_t some = __builtin_amdgcn_ballot_w64(s > 0.0), past = __builtin_amdgcn_ballot_w64(s > 0.0 && before + end > goal);
        if (past) {
            const int k = __builtin_ctzll(past);
            part = p0 + k;
            before += __shfl(end - s, k, 64);
        } else {
            if (some) {
                const int k = 63 - __builtin_clzll(some);
                last = p0 + k;
                last_before = before + __shfl(end - s, k, 64);
            }
            before += __shfl(end, 63, 64);
        }
    }
    if (part < 0) {
        part = last;
        before = last_before;
    }
    // a thread's kMine tokens of the part, the wave in which the sum passes, its thread, and the token
    constexpr int kMine = kPart / kWalkThreads;
    __shared__ double sums[kWalkThreads / 64];
    const int64_t base = (int64_t)part * kPart;
    const int m = (int)min((int64_t)kPart, io.V - base);
    double mine[kMine], s = 0.0;
#pragma unroll
    for (int e = 0; e < kMine; ++e) {
        const int at = tid * kMine + e;
        mine[e] = at < m ? weigh(w, per, base + at, b) : 0.0;
    }
    for (int j = 0; j < n_gone; ++j) {
        const int64_t at = token_of(gone_row(j)) - base - tid * kMine;
#pragma unroll
        for (int e = 0; e < kMine; ++e)
            if (at == e) mine[e] = 0.0;
    }
#pragma unroll
    for (int e = 0; e < kMine; ++e) s += mine[e];
    const double end = wave_prefix_sum(s);
    if (lane == 63) sums[tid >> 6] = end;
    __syncthreads();
    int who = -1, last_who = 0;
#pragma unroll
    for (int i = 0; i < kWalkThreads / 64; ++i) {
        if (who >= 0) continue;
        if (sums[i] > 0.0) last_who = i;
        if (sums[i] > 0.0 && before + sums[i] > goal) who = i;
        else before += sums[i];
    }
    const bool behind = who < 0;              // (roundings again: the last token of all)
    if ((tid >> 6) != (behind ? last_who : who)) return;
    const uint64_t some = __builtin_amdgcn_ballot_w64(s > 0.0), past = __builtin_amdgcn_ballot_w64(s > 0.0 && !behind && before + end > goal);
    if (lane != (past ? __builtin_ctzll(past) : 63 - __builtin_clzll(some | 1))) return;
    double sum = before + (end - s);
    int64_t token = -1;
#pragma unroll
    for (int e = 0; e < kMine; ++e) {
        if (!(mine[e] > 0.0) || (past && token >= 0 && sum > goal)) continue;
        token = base + tid * kMine + e;
        sum += mine[e];
    }
    io.next[slot] = token;
}

// Bytes of the workspace's lists, in the order of VerifyIo.
constexpr int64_t verify_ws(int64_t n_slots, int64_t rows, int64_t V) {
    const int64_t parts = (V + kPart - 1) / kPart;
    return rows * (parts + 1) * (int64_t)sizeof(RowPart) + rows * 12 + n_slots * (parts * 8 + (int64_t)sizeof(Wait));
}

}  // namespace
}  // namespace sx8

extern "C" int32_t sx8_draft_tree(const int32_t* parents, const int32_t* cu, int64_t n_slots, int64_t rows, int32_t words,
                                  uint64_t* mask, int32_t* depth, void* stream) {
    using namespace sx8;
    const char* what = "sx8_draft_tree";
    if (!cu || (rows > 0 && (!parents || !mask || !depth))) return fail(SX8_ERR_INVALID, "%s: null pointer", what);
    if (n_slots <= 0 || n_slots > kKv4MaxSlots || rows < 0 || rows > 0x7FFFFFFF || words < 1 || words > kMaxWords)
        return fail(SX8_ERR_INVALID, "%s: bad sizes (n_slots 1..%d, rows, words 1..%d)", what, kKv4MaxSlots, kMaxWords);
    if (!aligned(parents, 4) || !aligned(cu, 4) || !aligned(mask, 8) || !aligned(depth, 4))
        return fail(SX8_ERR_INVALID, "%s: parents, cu and depth must be 4-byte aligned, mask 8-byte", what);
    if (rows == 0) return ok();
    const Kv4Shape sh{(int)n_slots, 1, 1, 0, (int)rows};
    hipLaunchKernelGGL(k_draft_tree, dim3((unsigned)n_slots), dim3(256), 0, as_stream(stream), parents, cu, sh, words, mask, depth);
    return check_launch(what);
}

extern "C" int64_t sx8_draft_verify_workspace_bytes(int64_t n_slots, int64_t rows, int64_t V) {
    using namespace sx8;
    if (n_slots <= 0 || n_slots > kKv4MaxSlots || rows < 0 || rows > 1 << 22 || V <= 0 || V > 1 << 27) return -1;
    return verify_ws(n_slots, rows, V);
}

extern "C" int32_t sx8_draft_verify(const void* logits, int64_t logits_stride, int32_t dtype, const int64_t* tokens,
                                    const int32_t* parents, const int32_t* cu, int64_t n_slots, int64_t rows, int64_t V,
                                    const float* u, const float* temperature, float t, const void* probs,
                                    int64_t probs_stride, int32_t probs_dtype, int32_t* path, int32_t* counts, int64_t* next,
                                    void* workspace, int64_t workspace_bytes, void* stream) {
    return sx8_draft_verify_within(logits, logits_stride, dtype, tokens, parents, nullptr, cu, n_slots, rows, V, u, temperature, t,
                                   probs, probs_stride, probs_dtype, path, counts, next, workspace, workspace_bytes, stream);
}

extern "C" int32_t sx8_draft_verify_within(const void* logits, int64_t logits_stride, int32_t dtype, const int64_t* tokens,
                                           const int32_t* parents, const int32_t* depth, const int32_t* cu, int64_t n_slots,
                                           int64_t rows, int64_t V, const float* u, const float* temperature, float t,
                                           const void* probs, int64_t probs_stride, int32_t probs_dtype, int32_t* path,
                                           int32_t* counts, int64_t* next, void* workspace, int64_t workspace_bytes,
                                           void* stream) {
    using namespace sx8;
    const char* what = "sx8_draft_verify";
    if (!cu || !counts || !next || (rows > 0 && (!logits || !tokens || !parents || !path)))
        return fail(SX8_ERR_INVALID, "%s: null pointer", what);
    if (sx8_draft_verify_workspace_bytes(n_slots, rows, V) < 0)
        return fail(SX8_ERR_INVALID, "%s: bad sizes (n_slots 1..%d, rows up to 2^22, V 1..2^27)", what, kKv4MaxSlots);
    if (dtype < 0 || dtype > 2 || (probs && (probs_dtype < 0 || probs_dtype > 2)))
        return fail(SX8_ERR_INVALID, "%s: dtypes must be 0 (fp16), 1 (bf16) or 2 (float32)", what);
    const int64_t la = dtype == 2 ? 4 : 2, pa = probs_dtype == 2 ? 4 : 2;
    if (!aligned(logits, la) || !aligned(tokens, 8) || !aligned(parents, 4) || !aligned(depth, 4) || !aligned(cu, 4) || !aligned(u, 4) ||
        !aligned(temperature, 4) || !aligned(probs, pa) || !aligned(path, 4) || !aligned(counts, 4) || !aligned(next, 8))
        return fail(SX8_ERR_INVALID, "%s: pointers must be aligned to their values", what);
    if (logits_stride < V || logits_stride > (int64_t)1 << 40 || (probs && (probs_stride < V || probs_stride > (int64_t)1 << 40)))
        return fail(SX8_ERR_INVALID, "%s: row strides must be V or more", what);
    if (rows > 0 && !u && (temperature || t > 0.f)) return fail(SX8_ERR_INVALID, "%s: random numbers needed where a temperature is above zero", what);
    if (!workspace || workspace_bytes < verify_ws(n_slots, rows, V) || !aligned(workspace, 256))
        return fail(SX8_ERR_INVALID, "%s: workspace needs %lld bytes, 256-byte aligned", what, (long long)verify_ws(n_slots, rows, V));
    const int parts = (int)((V + kPart - 1) / kPart);
    VerifyIo io{logits, logits_stride, tokens, parents, cu, Kv4Shape{(int)n_slots, 1, 1, 0, (int)rows}, V, parts, u, temperature, t, depth,
                probs, probs_stride, path, counts, next, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr};
    io.part = reinterpret_cast<RowPart*>(workspace);
    io.row = io.part + rows * parts;
    io.p = reinterpret_cast<double*>(io.row + rows);
    io.wait = reinterpret_cast<Wait*>(io.p + rows);
    io.slot_sum = reinterpret_cast<double*>(io.wait + n_slots);
    io.gone = reinterpret_cast<int32_t*>(io.slot_sum + n_slots * parts);
    const bool wide = aligned(logits, 16) && logits_stride * la % 16 == 0;
    auto with = [&](auto ty) {
        constexpr int kType = decltype(ty)::value;
        const hipStream_t st = as_stream(stream);
        auto row = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3((unsigned)rows, (unsigned)parts), dim3(kRowThreads), 0, st, io); };
        auto walk = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3((unsigned)n_slots), dim3(kWalkThreads), 0, st, io); };
        if (rows > 0 && wide) row(k_verify_rows<kType, true>);
        else if (rows > 0) row(k_verify_rows<kType, false>);
        if (!probs) return walk(k_verify_walk<kType, -1, false>);
        auto drawn = [&](auto pt) {
            constexpr int kProbs = decltype(pt)::value;
            walk(k_verify_walk<kType, kProbs, false>);
            hipLaunchKernelGGL((k_verify_left<kType, kProbs>), dim3((unsigned)parts, (unsigned)n_slots), dim3(kRowThreads), 0, st, io);
            walk(k_verify_walk<kType, kProbs, true>);
        };
        if (probs_dtype == 0) drawn(std::integral_constant<int, 0>{});
        else if (probs_dtype == 1) drawn(std::integral_constant<int, 1>{});
        else drawn(std::integral_constant<int, 2>{});
    };
    if (dtype == 0) with(std::integral_constant<int, 0>{});
    else if (dtype == 1) with(std::integral_constant<int, 1>{});
    else with(std::integral_constant<int, 2>{});
    return check_launch(what);
}
