// sx8_kv4_dev.h -- device pieces shared by the kernels over packed sequences and the paged cache.
#pragma once
#include "sx8_device.h"
#include "sx8_kv4.h"

namespace sx8 {

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

// 16-bit value of dtype (fp16 or bf16) <-> float; rounding to nearest even.
template <bool kBf16>
__device__ __forceinline__ float ld16(uint32_t bits) {
    if constexpr (kBf16) return __builtin_bit_cast(float, bits << 16);
    else return sx8_h2f(bits);
}
template <bool kBf16>
__device__ __forceinline__ uint32_t st16(float v) {
    if constexpr (kBf16) return __builtin_bit_cast(uint16_t, (__bf16)v);
    else return __builtin_bit_cast(uint16_t, (_Float16)v);
}
// a | b << 16
template <bool kBf16>
__device__ __forceinline__ uint32_t pack16(float a, float b) {
    typedef float f2 __attribute__((ext_vector_type(2)));
    typedef _Float16 h2 __attribute__((ext_vector_type(2)));
    typedef __bf16 b2 __attribute__((ext_vector_type(2)));
    if constexpr (kBf16) return __builtin_bit_cast(uint32_t, __builtin_convertvector((f2{a, b}), b2));
    else return __builtin_bit_cast(uint32_t, __builtin_convertvector((f2{a, b}), h2));
}
__device__ __forceinline__ uint32_t half_of(uint32_t word, int i) { return i & 1 ? word >> 16 : word & 0xFFFFu; }

// A value that is the same in every lane, in scalar registers.
__device__ __forceinline__ int64_t uniform(int64_t v) {
    return (int64_t)((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(v >> 32)) << 32 |
                     (uint32_t)__builtin_amdgcn_readfirstlane((int)v));
}

__device__ __forceinline__ int64_t lane_of(int64_t v, int lane) {
    return (int64_t)((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), lane) << 32 |
                     (uint32_t)__builtin_amdgcn_readlane((int)v, lane));
}

template <int kCtrl>
__device__ __forceinline__ float dpp_lane(float v) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), kCtrl, 0xF, 0xF, false));
}

// Sum of v over the lanes up to this one: shifts within rows of 16 lanes, then each row's last lane to the rows above.
template <int kCtrl, int kRows>
__device__ __forceinline__ int64_t add_dpp(int64_t v) {
    const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)v, kCtrl, kRows, 0xF, false);
    const uint32_t hi = __builtin_amdgcn_update_dpp(0, (int)(v >> 32), kCtrl, kRows, 0xF, false);
    return v + (int64_t)((uint64_t)hi << 32 | lo);
}
__device__ __forceinline__ int64_t wave_prefix(int64_t v) {
    v = add_dpp<0x111, 0xF>(v);                      // row_shr 1, 2, 4, 8
    v = add_dpp<0x112, 0xF>(v);
    v = add_dpp<0x114, 0xF>(v);
    v = add_dpp<0x118, 0xF>(v);
    v = add_dpp<0x142, 0xA>(v);                      // row_bcast 15 into rows 1 and 3
    return add_dpp<0x143, 0xC>(v);                   // row_bcast 31 into rows 2 and 3
}

// Sum of v over the wave, in a scalar register.
__device__ __forceinline__ int wave_sum(int v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);
    return __builtin_amdgcn_readlane(v, 63);
}

// Prefix sums of f(s) over n items into pre[0 .. n] (LDS), every thread of the work-group (kT threads) taking part.
template <int kT, typename P, typename F>
__device__ __forceinline__ void prefix_sums(int n, P* pre, F&& f) {
    __shared__ int64_t wsum[kT / 64];
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
    int64_t base = 0;
    if (tid == 0) pre[0] = 0;
    for (int s0 = 0; s0 < n; s0 += kT) {
        const int64_t v = wave_prefix(s0 + tid < n ? f(s0 + tid) : 0);
        if (lane == 63) wsum[w] = v;
        __syncthreads();
        int64_t before = base, all = base;
#pragma unroll
        for (int i = 0; i < kT / 64; ++i) {
            if (i < w) before += wsum[i];
            all += wsum[i];
        }
        if (s0 + tid < n) pre[s0 + tid + 1] = (P)(before + v);
        base = all;
        __syncthreads();
    }
}

// The item whose range of the prefix sums holds x (pre[0] <= x < pre[n]); every thread gets it.
template <int kT>
__device__ __forceinline__ int find_item(int n, const int64_t* pre, int64_t x) {
    __shared__ int found;
    for (int s = threadIdx.x; s < n; s += kT)
        if (pre[s] <= x && x < pre[s + 1]) found = s;
    __syncthreads();
    return __builtin_amdgcn_readfirstlane(found);
}

}  // namespace sx8
