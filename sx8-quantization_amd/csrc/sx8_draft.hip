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
// parts of kPart logits; then a work-group for each slot walks its tree, where a test needs one logit, and draws the next token, where
// the parts' sums say in which part it lies.  All in binary64: a token must not depend on the order in which 150000 weights
// were added, and a border of the cumulated sum lies within a binary32 rounding of u once in some hundred draws.
constexpr int kPart = 8192, kThreads = 256;

struct RowPart {
    double sum;                           // of exp((x - top) / temperature), or 0 (greedy)
    float top;                            // largest logit of the part (-infinity: none)
    int32_t arg;                          // its first index
};
static_assert(sizeof(RowPart) == 16, "part");

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
    const void* probs;
    int64_t probs_stride;
    int32_t *path, *counts;
    int64_t* next;
    RowPart* part;                        // [rows][parts]
    int64_t* gone;                        // [rows]: tokens of a slot that are out of p at its current row
    double* slot_sum;                     // [n_slots][parts]: sums of what is left of p
};

template <int kType>                      // 0 fp16, 1 bf16, 2 float32; NaN: -infinity
__device__ __forceinline__ float value(const void* base, int64_t at) {
    if constexpr (kType == 2) return static_cast<const float*>(base)[at];
    else return ld16<kType == 1>(static_cast<const uint16_t*>(base)[at]);
}
__device__ __forceinline__ float logit(float x) { return x == x ? x : -__builtin_inff(); }

// exp((x - top) / temperature): 1 for the largest (an infinity too)
__device__ __forceinline__ double weight(float x, float top, double scale) {
    return x == top ? 1.0 : x - top == -__builtin_inff() ? 0.0 : exp(((double)x - (double)top) * scale);
}
__device__ __forceinline__ float temperature_of(const VerifyIo& io, int slot) { return io.temperature ? io.temperature[slot] : io.t; }

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
// The sum over the work-group, the same in every thread.
__device__ __forceinline__ double group_add(double v) {
    __shared__ double s[kThreads / 64];
    v = wave_add(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = v;
    __syncthreads();
    double r = 0.0;
#pragma unroll
    for (int i = 0; i < kThreads / 64; ++i) r += s[i];
    return r;
}
// (top, first index) of two candidates
__device__ __forceinline__ void better(float& top, int& arg, float t, int a) {
    if (t > top || (t == top && a < arg)) {
        top = t;
        arg = a;
    }
}

// The slot that has row r, or -1.
__device__ __forceinline__ int slot_of(const Kv4Shape& sh, const int32_t* cu, int r) {
    const int lane = threadIdx.x & 63;
    // (ends grow: the slots that end at or before r come first; 64 at a time)
    int s = 0;
    for (; s < sh.n_slots; s += 64) {
        const int at = s + lane;
        const uint64_t before = __builtin_amdgcn_ballot_w64(at < sh.n_slots && cu[at + 1] <= r);
        const int k = __builtin_popcountll(before);
        if (k < 64) {
            s += k;
            break;
        }
    }
    if (s >= sh.n_slots || cu[s] > r) return -1;
    return s;
}

template <int kType>
__global__ __launch_bounds__(kThreads) void k_verify_rows(const VerifyIo io) {
    constexpr int kE = kPart / kThreads;
    const int r = blockIdx.x, part = blockIdx.y, tid = threadIdx.x, lane = tid & 63;
    const int slot = slot_of(io.sh, io.cu, r);
    if (slot < 0) return;
    const int64_t base = (int64_t)part * kPart;
    const int n = (int)min((int64_t)kPart, io.V - base);
    float x[kE], top = -__builtin_inff();
    int arg = 0x7FFFFFFF;
#pragma unroll
    for (int i = 0; i < kE; ++i) {
        const int at = tid + kThreads * i;
        x[i] = at < n ? logit(value<kType>(io.logits, r * io.stride + base + at)) : -__builtin_inff();
    }
#pragma unroll
    for (int i = 0; i < kE; ++i)
        if (x[i] > top) {
            top = x[i];
            arg = (int)base + tid + kThreads * i;
        }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) better(top, arg, __shfl_xor(top, o, 64), __shfl_xor(arg, o, 64));
    __shared__ float tops[kThreads / 64];
    __shared__ int args[kThreads / 64];
    if (lane == 0) {
        tops[tid >> 6] = top;
        args[tid >> 6] = arg;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kThreads / 64; ++i) better(top, arg, tops[i], args[i]);
    const float temp = temperature_of(io, slot);
    double sum = 0.0;
    if (temp > 0.f && top > -__builtin_inff()) {
        const double scale = 1.0 / (double)temp;
#pragma unroll
        for (int i = 0; i < kE; ++i) sum += weight(x[i], top, scale);
        sum = group_add(sum);
    }
    if (tid == 0) io.part[(int64_t)r * io.parts + part] = RowPart{sum, top, arg};
}

// The largest logit of a row, its first index and the sum of its weights (wave-wide; every lane gets them).
struct RowSum {
    double sum;
    float top;
    int arg;
};
__device__ __forceinline__ RowSum row_sum(const VerifyIo& io, int64_t row, bool greedy, double scale) {
    const int lane = threadIdx.x & 63;
    const RowPart* const p = io.part + row * io.parts;
    RowSum r = {0.0, -__builtin_inff(), 0x7FFFFFFF};
    for (int i = lane; i < io.parts; i += 64) better(r.top, r.arg, p[i].top, p[i].arg);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) better(r.top, r.arg, __shfl_xor(r.top, o, 64), __shfl_xor(r.arg, o, 64));
    if (!greedy)
        for (int i = lane; i < io.parts; i += 64)
            if (p[i].top > -__builtin_inff()) r.sum += p[i].sum * weight(p[i].top, r.top, scale);
    r.sum = wave_add(r.sum);
    return r;
}

// What is left of p at a row: weights max(a w(x) / sum - b q(x), 0), without the tokens in `gone`.
template <int kType, int kProbs>          // kProbs -1: no draft probabilities
__global__ __launch_bounds__(kThreads) void k_verify_walk(const VerifyIo io) {
    __shared__ double sums[kThreads];
    const int slot = blockIdx.x, tid = threadIdx.x, lane = tid & 63;
    int first, n;
    kv4_rows(io.sh, io.cu, slot, &first, &n);
    if (n == 0) {
        if (tid == 0) {
            io.counts[slot] = 0;
            io.next[slot] = -1;
        }
        return;
    }
    for (int i = tid; i < n; i += kThreads) io.path[first + i] = i == 0 ? 0 : -1;
    const float temp = temperature_of(io, slot);
    const bool greedy = !(temp > 0.f);
    const double scale = greedy ? 0.0 : 1.0 / (double)temp;
    __syncthreads();
    int64_t* const gone = io.gone + first;
    // the walk: every wave does it alike
    int cur = 0, count = 1, n_gone = 0;
    double left = 1.0, a = 1.0, b = 0.0;
    RowSum rs = row_sum(io, first, greedy, scale);
    double* const slot_sum = io.slot_sum + (int64_t)slot * io.parts;
    // the weight that is left of token x at the current row, of coefficients ca, cb
    auto weigh = [&](int64_t x, double ca, double cb) -> double {
        const float l = logit(value<kType>(io.logits, ((int64_t)first + cur) * io.stride + x));
        double v = rs.top > -__builtin_inff() ? weight(l, rs.top, scale) / rs.sum : 0.0;
        if constexpr (kProbs >= 0) {
            if (cb != 0.0) v = fmax(ca * v - cb * (double)value<kProbs < 0 ? 0 : kProbs>(io.probs, ((int64_t)first + cur) * io.probs_stride + x), 0.0);
        }
        return v;
    };
    auto is_gone = [&](int64_t x) {
        for (int i = 0; i < n_gone; ++i)
            if (gone[i] == x) return true;
        return false;
    };
    double total = 1.0;                    // of the weights of coefficients a, b
    for (int i0 = 0; i0 < n; i0 += 64) {
        const int row = i0 + lane;
        const int par = row < n && row > 0 ? io.parents[first + row] : -1;
        const int64_t tok = row < n ? io.tokens[first + row] : -1;
        const float un = row < n && io.u ? io.u[first + row] : 0.f;
        uint64_t todo = __builtin_amdgcn_ballot_w64(par == cur);
        while (todo) {
            const int k = __builtin_ctzll(todo);
            todo &= todo - 1;
            const int64_t x = lane_of(tok, k);
            const double uk = (double)__builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, un), k));
            const bool in = x >= 0 && x < io.V;
            bool keep;
            if (greedy) {
                keep = in && rs.top > -__builtin_inff() && x == rs.arg;
            } else if constexpr (kProbs < 0) {
                const double p = in && !is_gone(x) ? weigh(x, 1.0, 0.0) : 0.0;
                keep = p > 0.0 && uk < 1.0 && uk * left < p;
                if (!keep && p > 0.0) {
                    __syncthreads();
                    if (tid == 0) gone[n_gone] = x;
                    __syncthreads();
                    ++n_gone;
                    left -= p;
                }
            } else {
                const double p = in ? weigh(x, a, b) / total : 0.0;
                const double q = in ? (double)value<kProbs>(io.probs, ((int64_t)first + cur) * io.probs_stride + x) : 0.0;
                keep = p > 0.0 && uk * q < p;
                if (!keep && in && rs.top > -__builtin_inff()) {
                    // max(p - q, 0) with p = max(a w - b q, 0) / total: coefficients a / total and b / total + 1
                    const double na = a / total, nb = b / total + 1.0;
                    double all = 0.0;
                    for (int part = 0; part < io.parts; ++part) {
                        double s = 0.0;
                        const int64_t base = (int64_t)part * kPart, m = min((int64_t)kPart, io.V - base);
                        for (int e = tid; e < m; e += kThreads) s += weigh(base + e, na, nb);
                        s = group_add(s);
                        if (tid == 0) slot_sum[part] = s;
                        all += s;
                    }
                    a = na;
                    b = nb;
                    total = all;
                    if (!(all > 0.0)) {
                        a = total = 1.0;
                        b = 0.0;
                    }
                }
            }
            if (keep) {
                cur = i0 + k;
                if (tid == 0) io.path[first + count] = cur;
                ++count;
                n_gone = 0;
                left = a = total = 1.0;
                b = 0.0;
                rs = row_sum(io, (int64_t)first + cur, greedy, scale);
                todo = __builtin_amdgcn_ballot_w64(par == cur && lane > k);
            }
        }
    }
    if (tid == 0) io.counts[slot] = count;
    if (greedy || !(rs.top > -__builtin_inff())) {
        if (tid == 0) io.next[slot] = rs.top > -__builtin_inff() ? rs.arg : -1;
        return;
    }
    // the sums of the parts of what is left
    const RowPart* const rp = io.part + ((int64_t)first + cur) * io.parts;
    auto left_of = [&](int64_t x) { return is_gone(x) ? 0.0 : weigh(x, a, b); };
    if (b == 0.0) {
        for (int i = tid; i < io.parts; i += kThreads)
            slot_sum[i] = rp[i].top > -__builtin_inff() ? rp[i].sum * weight(rp[i].top, rs.top, scale) / rs.sum : 0.0;
        __syncthreads();
        for (int i = 0; i < n_gone; ++i) {
            const int part = (int)(gone[i] / kPart);
            double s = 0.0;
            const int64_t base = (int64_t)part * kPart, m = min((int64_t)kPart, io.V - base);
            for (int e = tid; e < m; e += kThreads) s += left_of(base + e);
            s = group_add(s);
            if (tid == 0) slot_sum[part] = s;
        }
        __syncthreads();
        double s = 0.0;
        for (int i = tid; i < io.parts; i += kThreads) s += slot_sum[i];
        total = group_add(s);
        if (!(total > 0.0)) {                 // nothing left: the target's own
            n_gone = 0;
            for (int i = tid; i < io.parts; i += kThreads)
                slot_sum[i] = rp[i].top > -__builtin_inff() ? rp[i].sum * weight(rp[i].top, rs.top, scale) / rs.sum : 0.0;
            __syncthreads();
            s = 0.0;
            for (int i = tid; i < io.parts; i += kThreads) s += slot_sum[i];
            total = group_add(s);
        }
    }
    __syncthreads();
    // the part in which the sum passes u * total (or, by roundings, the last one that has any)
    const double goal = (io.u ? (double)io.u[first] : 0.0) * total;
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
    // a thread's kMine tokens of the part, then the tokens of the thread in which the sum passes
    constexpr int kMine = kPart / kThreads;
    const int64_t base = (int64_t)part * kPart;
    const int m = (int)min((int64_t)kPart, io.V - base);
    double mine = 0.0;
    for (int e = tid * kMine; e < min(m, (tid + 1) * kMine); ++e) mine += left_of(base + e);
    sums[tid] = mine;
    __syncthreads();
    int64_t who = -1, last_who = 0;
    for (int t0 = 0; t0 < kThreads && who < 0; t0 += 64) {
        const double s = sums[t0 + lane], end = wave_prefix_sum(s);
        const uint64_t some = __builtin_amdgcn_ballot_w64(s > 0.0), past = __builtin_amdgcn_ballot_w64(s > 0.0 && before + end > goal);
        if (past) {
            const int k = __builtin_ctzll(past);
            who = t0 + k;
            before += __shfl(end - s, k, 64);
        } else {
            if (some) last_who = t0 + 63 - __builtin_clzll(some);
            before += __shfl(end, 63, 64);
        }
    }
    const bool behind = who < 0;              // (roundings again: the last token of all)
    if (behind) who = last_who;
    static_assert(kMine <= 64, "a wave");
    const int e = (int)who * kMine + lane;
    const double s = lane < kMine && e < m ? left_of(base + e) : 0.0, end = wave_prefix_sum(s);
    const uint64_t some = __builtin_amdgcn_ballot_w64(s > 0.0), past = __builtin_amdgcn_ballot_w64(s > 0.0 && !behind && before + end > goal);
    if (tid == 0) io.next[slot] = base + who * kMine + (past ? __builtin_ctzll(past) : 63 - __builtin_clzll(some | 1));
}

constexpr int64_t verify_ws(int64_t n_slots, int64_t rows, int64_t V) {
    const int64_t parts = (V + kPart - 1) / kPart;
    return rows * (parts * (int64_t)sizeof(RowPart) + 8) + n_slots * parts * 8;
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
    if (n_slots <= 0 || n_slots > kKv4MaxSlots || rows < 0 || rows > 1 << 22 || V <= 0 || V > 1 << 28) return -1;
    return verify_ws(n_slots, rows, V);
}

extern "C" int32_t sx8_draft_verify(const void* logits, int64_t logits_stride, int32_t dtype, const int64_t* tokens,
                                    const int32_t* parents, const int32_t* cu, int64_t n_slots, int64_t rows, int64_t V,
                                    const float* u, const float* temperature, float t, const void* probs,
                                    int64_t probs_stride, int32_t probs_dtype, int32_t* path, int32_t* counts, int64_t* next,
                                    void* workspace, int64_t workspace_bytes, void* stream) {
    using namespace sx8;
    const char* what = "sx8_draft_verify";
    if (!cu || !counts || !next || (rows > 0 && (!logits || !tokens || !parents || !path)))
        return fail(SX8_ERR_INVALID, "%s: null pointer", what);
    if (sx8_draft_verify_workspace_bytes(n_slots, rows, V) < 0)
        return fail(SX8_ERR_INVALID, "%s: bad sizes (n_slots 1..%d, rows up to 2^22, V 1..2^28)", what, kKv4MaxSlots);
    if (dtype < 0 || dtype > 2 || (probs && (probs_dtype < 0 || probs_dtype > 2)))
        return fail(SX8_ERR_INVALID, "%s: dtypes must be 0 (fp16), 1 (bf16) or 2 (float32)", what);
    const int64_t la = dtype == 2 ? 4 : 2, pa = probs_dtype == 2 ? 4 : 2;
    if (!aligned(logits, la) || !aligned(tokens, 8) || !aligned(parents, 4) || !aligned(cu, 4) || !aligned(u, 4) ||
        !aligned(temperature, 4) || !aligned(probs, pa) || !aligned(path, 4) || !aligned(counts, 4) || !aligned(next, 8))
        return fail(SX8_ERR_INVALID, "%s: pointers must be aligned to their values", what);
    if (logits_stride < V || logits_stride > (int64_t)1 << 40 || (probs && (probs_stride < V || probs_stride > (int64_t)1 << 40)))
        return fail(SX8_ERR_INVALID, "%s: row strides must be V or more", what);
    if (!u && (temperature || t > 0.f)) return fail(SX8_ERR_INVALID, "%s: random numbers needed where a temperature is above zero", what);
    if (!workspace || workspace_bytes < verify_ws(n_slots, rows, V) || !aligned(workspace, 256))
        return fail(SX8_ERR_INVALID, "%s: workspace needs %lld bytes, 256-byte aligned", what, (long long)verify_ws(n_slots, rows, V));
    const int parts = (int)((V + kPart - 1) / kPart);
    VerifyIo io{logits, logits_stride, tokens, parents, cu, Kv4Shape{(int)n_slots, 1, 1, 0, (int)rows}, V, parts, u, temperature, t,
                probs, probs_stride, path, counts, next, nullptr, nullptr, nullptr};
    io.part = reinterpret_cast<RowPart*>(workspace);
    io.gone = reinterpret_cast<int64_t*>(io.part + rows * parts);
    io.slot_sum = reinterpret_cast<double*>(io.gone + rows);
    auto with = [&](auto ty) {
        constexpr int kType = decltype(ty)::value;
        if (rows > 0)
            hipLaunchKernelGGL((k_verify_rows<kType>), dim3((unsigned)rows, (unsigned)parts), dim3(kThreads), 0, as_stream(stream), io);
        auto walk = [&](auto kernel) {
            hipLaunchKernelGGL(kernel, dim3((unsigned)n_slots), dim3(kThreads), 0, as_stream(stream), io);
        };
        if (!probs) walk(k_verify_walk<kType, -1>);
        else if (probs_dtype == 0) walk(k_verify_walk<kType, 0>);
        else if (probs_dtype == 1) walk(k_verify_walk<kType, 1>);
        else walk(k_verify_walk<kType, 2>);
    };
    if (dtype == 0) with(std::integral_constant<int, 0>{});
    else if (dtype == 1) with(std::integral_constant<int, 1>{});
    else with(std::integral_constant<int, 2>{});
    return check_launch(what);
}
