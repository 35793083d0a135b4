// The router's choice: the k experts of the largest logits of each token and their weights, and the gradient.
//   chosen   ties go to the lowest index; logits of -inf and NaN are masked, never chosen and without a share in any sum;
//            a choice with nothing left has index -1 and weight 0
//   softmax  w_j = scale exp(l_j - m) / sum_i exp(l_i - m), i over all unmasked experts, or over the chosen (normalize)
//   sigmoid  w_j = scale s(l_j), or scale s(l_j) / sum over the chosen (normalize): the softmax of log s, which cannot
//            divide zero by zero however low the logits
// A warp keeps a row in registers (one read of the logits) and takes the largest value k times.  Values stand as unsigned
// keys in the order of the values, so the choice is exact; 16-bit logits share a word with their index, which makes keys
// differ and one redux.sync say both.  What is chosen is never removed: the next largest is the largest below it, which one
// addition and maximum a value finds (8192 x 256 bf16, k = 8: removing 11.1 us, this 6.7; f32, where equal values want a second
// look at the lane's, 11.9).  Sums are held in 32 bits.
#include <algorithm>
#include <climits>
#include <type_traits>

#include "launch.h"
#include "token_rows.cuh"

namespace qmm {

namespace {

constexpr int WARPS = 4; // rows per CTA

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

template <typename T, int PER_LANE>
__global__ void __launch_bounds__(WARPS * 32) route_kernel(const __grid_constant__ RouteArgs a) {
    ptx::grid_dependency_wait();
    constexpr int V = PER_LANE * sizeof(T) < 16 ? PER_LANE : 16 / (int)sizeof(T); // neighbours that a lane reads at once
    const int lane = threadIdx.x & 31;
    const int64_t t = (int64_t)blockIdx.x * WARPS + threadIdx.x / 32;
    if (t >= a.tokens) return;
    const T *row = (const T *)a.logits + t * a.logits_ld;
    auto expert = [&](int i) { return i / V * (32 * V) + lane * V + i % V; }; // of the lane's value i
    T raw[PER_LANE];
    if (a.aligned) { // rows start on, and hold a multiple of, V values
        struct alignas(V * sizeof(T)) Group { T v[V]; };
#pragma unroll
        for (int i = 0; i < PER_LANE; i += V)
            if (expert(i) < a.experts) {
                const Group g = *reinterpret_cast<const Group *>(row + expert(i));
#pragma unroll
                for (int j = 0; j < V; ++j) raw[i + j] = g.v[j];
            }
    } else {
#pragma unroll
        for (int i = 0; i < PER_LANE; ++i)
            if (expert(i) < a.experts) raw[i] = row[expert(i)];
    }
    uint32_t key[PER_LANE];
#pragma unroll
    for (int i = 0; i < PER_LANE; ++i) {
        key[i] = expert(i) < a.experts ? order_key(to_f32(raw[i])) : 0u;
        // the value's bits are the upper 16 of its key (bf16) or of its own (f16)
        if constexpr (sizeof(T) == 2) {
            if constexpr (std::is_same<T, __half>::value) {
                const uint32_t u = __half_as_ushort(raw[i]), k = (u & 0x7fffu) == 0 ? 0x8000u : u & 0x8000u ? ~u & 0xffffu : u | 0x8000u;
                key[i] = key[i] ? k << 16 : 0u;
            }
            key[i] = key[i] ? (key[i] & 0xffff0000u) | (0xffffu - expert(i)) : 0u;
        }
    }
    auto value = [&](uint32_t k) { // of a key
        if constexpr (std::is_same<T, __half>::value) {
            const uint32_t u = k >> 16;
            return fminf(__half2float(__ushort_as_half((unsigned short)(u & 0x8000u ? u & 0x7fffu : ~u))), LARGEST<T>);
        } else {
            return key_value<T>(sizeof(T) == 2 ? (k & 0x80000000u ? k & 0xffff0000u : k | 0xffffu) : k);
        }
    };
    uint32_t best = 0;
#pragma unroll
    for (int i = 0; i < PER_LANE; ++i) best = max(best, key[i]);
    float sum = 0.f, top = 0.f;
    if (a.scoring == SCORING_SOFTMAX && !a.normalize) {
        top = value(__reduce_max_sync(0xffffffffu, best));
#pragma unroll
        for (int i = 0; i < PER_LANE; ++i) sum += key[i] ? expf(fminf(to_f32(raw[i]), LARGEST<T>) - top) : 0.f;
        sum = warp_sum(sum);
    }
    uint32_t mine = 0; // key and index of choice `lane`
    int index = -1;
    if constexpr (sizeof(T) == 2) {
        for (int j = 0; j < a.choices; ++j) {
            const uint32_t most = __reduce_max_sync(0xffffffffu, best);
            if (most == 0) break;
            if (lane == j) mine = most;
            best = next_below(key, most);
        }
        if (mine) index = 0xffff - (int)(mine & 0xffffu);
    } else {
        for (int j = 0; j < a.choices;) {
            const uint32_t most = __reduce_max_sync(0xffffffffu, best);
            if (most == 0) break;
            uint32_t equal = 0; // the lane's values with this key, lowest index first
            if (best == most) {
#pragma unroll
                for (int i = 0; i < PER_LANE; ++i) equal |= key[i] == most ? 1u << i : 0u;
            }
            for (; j < a.choices; ++j) {
                const int i = __ffs(equal) - 1, own = equal ? expert(i) : INT_MAX, at = __reduce_min_sync(0xffffffffu, own);
                if (at == INT_MAX) break;
                if (own == at) equal &= equal - 1;
                if (lane == j) {
                    mine = most;
                    index = at;
                }
            }
            best = next_below(key, most);
        }
    }
    const bool chosen = index >= 0;
    float w;
    if (a.scoring == SCORING_SOFTMAX) {
        if (a.normalize) top = value(__shfl_sync(0xffffffffu, mine, 0)); // the first choice is the largest
        w = chosen ? expf(value(mine) - top) : 0.f;
        if (a.normalize) sum = warp_sum(w);
        w = chosen ? w / sum : 0.f;
    } else if (a.normalize) {
        const float l = chosen ? log_sigmoid(value(mine)) : -INFINITY;
        const float m = __shfl_sync(0xffffffffu, l, 0);
        w = chosen ? expf(l - m) : 0.f;
        sum = warp_sum(w);
        w = chosen ? w / sum : 0.f;
    } else {
        w = chosen ? sigmoid(value(mine)) : 0.f;
    }
    if (lane < a.choices) {
        a.weights[t * a.weights_ld + lane] = w * a.scale;
        a.indices[t * a.indices_ld + lane] = index;
    }
}

// Gradient of the logits.  With g the weights' gradient times scale:
//   softmax            dl_i = p_i (g_i - sum_j g_j p_j), over all experts; normalize: over the chosen, zero elsewhere
//   sigmoid            dl_j = g_j s_j (1 - s_j); normalize, q_j = s_j / sum: dl_j = q_j (1 - s_j) (g_j - sum_i g_i q_i)
// Lane j works on choice j; only the first form needs the logits of the experts that were not chosen.
template <typename T>
__global__ void __launch_bounds__(WARPS * 32) route_backward_kernel(const __grid_constant__ RouteArgs a) {
    extern __shared__ float shared[];
    ptx::grid_dependency_wait();
    const int lane = threadIdx.x & 31;
    const int64_t t = (int64_t)blockIdx.x * WARPS + threadIdx.x / 32;
    if (t >= a.tokens) return;
    float *grad = shared + threadIdx.x / 32 * a.experts;
    const T *row = (const T *)a.logits + t * a.logits_ld;
    T *out = (T *)a.diff_logits + t * a.diff_logits_ld;
    int index = lane < a.choices ? a.indices[t * a.indices_ld + lane] : -1;
    uint32_t key = (unsigned)index < (unsigned)a.experts ? order_key(to_f32(row[index])) : 0u;
    const bool chosen = key != 0;
    const float l = key_value<T>(key);
    float g = chosen ? a.weights[t * a.weights_ld + lane] * a.scale : 0.f;
    const bool dense = a.scoring == SCORING_SOFTMAX && !a.normalize;
    float top = 0.f, inverse = 0.f, inner = 0.f, d;
    for (int e = lane; e < a.experts; e += 32) grad[e] = 0.f;
    if (dense) {
        float m = -INFINITY, sum = 0.f;
        for (int e = lane; e < a.experts; e += 32) {
            const uint32_t k = order_key(to_f32(row[e]));
            if (k) m = fmaxf(m, key_value<T>(k));
        }
        top = warp_max(m);
        for (int e = lane; e < a.experts; e += 32) {
            const uint32_t k = order_key(to_f32(row[e]));
            if (k) sum += expf(key_value<T>(k) - top);
        }
        inverse = 1.f / warp_sum(sum); // (unused where every expert is masked)
        const float p = chosen ? expf(l - top) * inverse : 0.f;
        inner = warp_sum(g * p);
        d = g * p; // and - p * inner below, with all the others
    } else if (a.scoring == SCORING_SOFTMAX) {
        top = warp_max(chosen ? l : -INFINITY);
        const float e = chosen ? expf(l - top) : 0.f;
        const float sum = warp_sum(e), q = chosen ? e / sum : 0.f;
        d = q * (g - warp_sum(g * q));
    } else if (a.normalize) {
        const float ls = chosen ? log_sigmoid(l) : -INFINITY;
        const float m = warp_max(ls);
        const float e = chosen ? expf(ls - m) : 0.f;
        const float sum = warp_sum(e), q = chosen ? e / sum : 0.f;
        d = q * sigmoid(-l) * (g - warp_sum(g * q));
    } else {
        d = g * sigmoid(l) * sigmoid(-l);
    }
    __syncwarp();
    if (chosen) atomicAdd(&grad[index], d); // the choices of a row differ; a caller's own may not
    __syncwarp();
    for (int e = lane; e < a.experts; e += 32) {
        float v = grad[e];
        if (dense) {
            const uint32_t k = order_key(to_f32(row[e]));
            if (k) v -= expf(key_value<T>(k) - top) * inverse * inner;
        }
        out[e] = from_f32<T>(v);
    }
}

template <typename T> int launch_typed(const RouteArgs &a, bool backward, cudaStream_t st) {
    const int64_t grid = (a.tokens + WARPS - 1) / WARPS;
    if (grid > 0x7fffffff) return 3;
    int rc;
    if (backward) {
        rc = launch_dependent(route_backward_kernel<T>, a, (unsigned)grid, WARPS * 32, WARPS * a.experts * sizeof(float), st);
    } else {
        RouteArgs r = a;
        const int per_lane = a.experts <= 64 ? 2 : a.experts <= 128 ? 4 : a.experts <= 256 ? 8 : a.experts <= 512 ? 16 : 32;
        const int bytes = std::min(per_lane * (int)sizeof(T), 16), values = bytes / (int)sizeof(T);
        r.aligned = (uintptr_t)a.logits % bytes == 0 && a.experts % values == 0 && (a.tokens == 1 || a.logits_ld % values == 0);
        void (*kernel)(RouteArgs) = per_lane == 2 ? route_kernel<T, 2>
                : per_lane == 4                   ? route_kernel<T, 4>
                : per_lane == 8                   ? route_kernel<T, 8>
                : per_lane == 16                  ? route_kernel<T, 16>
                                                  : route_kernel<T, 32>;
        rc = launch_dependent(kernel, r, (unsigned)grid, WARPS * 32, 0, st);
    }
    if (rc == 0) count_launch();
    return rc;
}

int launch_any(const RouteArgs &a, bool backward, cudaStream_t st) {
    if (a.tokens == 0) return 0;
    switch (a.dt) {
        case DT_F32: return launch_typed<float>(a, backward, st);
        case DT_BF16: return launch_typed<__nv_bfloat16>(a, backward, st);
        case DT_F16: return launch_typed<__half>(a, backward, st);
        default: return 3;
    }
}

} // namespace

int launch_route(const RouteArgs &a, cudaStream_t st) { return launch_any(a, false, st); }
int launch_route_backward(const RouteArgs &a, cudaStream_t st) { return launch_any(a, true, st); }

} // namespace qmm
