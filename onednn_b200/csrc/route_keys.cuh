// What the router's kernels share: values as unsigned keys in the order of the values, and sums over a warp.
#pragma once
#include <type_traits>

#include "token_rows.cuh"

namespace qmm {

// Bits in the order of the values; -0 as +0; 0 for a masked value.
__device__ __forceinline__ uint32_t order_key(float v) {
    const uint32_t u = __float_as_uint(v + 0.f);
    const uint32_t k = u & 0x80000000u ? ~u : u | 0x80000000u;
    return v > -INFINITY ? k : 0u; // (false for a NaN too)
}
// +inf counts as the largest finite value of the logits' type, in the choice's weights and in their gradient alike.
template <typename T>
constexpr float LARGEST = std::is_same<T, __half>::value ? 65504.f : std::is_same<T, __nv_bfloat16>::value ? 3.38953139e38f : 3.402823466e38f;
template <typename T> __device__ __forceinline__ float key_value(uint32_t k) {
    return fminf(__uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k), LARGEST<T>);
}
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int s = 16; s > 0; s /= 2) v += __shfl_xor_sync(0xffffffffu, v, s);
    return v;
}
__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
    for (int s = 16; s > 0; s /= 2) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, s));
    return v;
}
__device__ __forceinline__ float sigmoid(float x) { return 1.f / (1.f + expf(-x)); }
__device__ __forceinline__ float log_sigmoid(float x) { return fminf(x, 0.f) - log1pf(expf(-fabsf(x))); }

// The largest key below `most`, 0 if there is none: key - most wraps for those below, beyond any difference of the others,
// and the largest wrapped difference is the nearest.
template <int N> __device__ __forceinline__ uint32_t next_below(const uint32_t (&key)[N], uint32_t most) {
    uint32_t d = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) d = max(d, key[i] - most);
    const uint32_t next = d + most;
    return next < most ? next : 0u;
}

} // namespace qmm
