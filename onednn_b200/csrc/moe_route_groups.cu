// The router's choice by score and bias, within the best groups of experts.
//   score    s = softmax or sigmoid of the logits, as moe_route.cu has them
//   chosen   the k largest of c = s + bias among the experts of the kept groups, which are those whose group_best (1 or 2)
//            largest c have the largest sum; ties go to the lowest group and expert
//   weights  of the chosen, from their scores without the bias
//   masked   logits of -inf and NaN as in moe_route.cu; an expert whose bias is -inf or NaN is never chosen, but counts in a
//            softmax's sum; +inf counts as the largest finite value of its type
// The choice is by the values of c in 64 bits.  32 bits say the same wherever the values that the choice falls between differ by
// more than what rounding can have moved them (8192 x 256: all but some 0.5 % of the rows); only the other rows are
// computed again in 64 bits, out of line.  So a warp keeps a row's c as 32-bit keys in registers, as moe_route.cu does, with the
// number of the value in the lane in the lowest bits: keys of a lane differ, and a redux and a ballot say which expert it is.
// Groups are looked at by 32 / groups lanes each, from shared memory.
#include <algorithm>

#include "launch.h"
#include "route_keys.cuh"

namespace qmm {

namespace {

constexpr int WARPS = 4; // rows per CTA

// words of shared memory between two groups: the lanes that look at different groups read different banks
__host__ __device__ inline int group_stride(int size, int lanes) { return (size + 31) / 32 * 32 + lanes; }
// lanes that look at one group together
__host__ __device__ inline int group_lanes(int groups) {
    int lanes = 32;
    while (lanes * groups > 32) lanes /= 2;
    return lanes;
}

// Relative error of a score in 32 bits, an upper bound.  A sigmoid: an exponential (2 units of 2^-23), a sum, a quotient.  A
// softmax: the argument is off by 2^-24 of itself, which is at most 104 where the exponential is not zero; its sum has at most
// 32 + 5 roundings, the exponential and the quotient are as above.
__device__ __forceinline__ float score_error(int scoring) { return scoring == SCORING_SIGMOID ? 0x1p-21f : 0x1p-16f; }

// The k choices of a row in 64 bits.  values: [experts] of this warp's own.  Lane j returns choice j, -1 without one.
template <typename T>
__device__ __noinline__ int choose_in_64_bits(const RouteArgs &a, const T *row, double *values) {
    const int lane = threadIdx.x & 31;
    const double none = -__longlong_as_double(0x7ff0000000000000ll);
    double top = none, sum = 0;
    if (a.scoring == SCORING_SOFTMAX) {
        for (int e = lane; e < a.experts; e += 32) {
            const uint32_t k = order_key(to_f32(row[e]));
            if (k) top = fmax(top, (double)key_value<T>(k));
        }
#pragma unroll
        for (int s = 16; s > 0; s /= 2) top = fmax(top, __shfl_xor_sync(0xffffffffu, top, s));
        for (int e = lane; e < a.experts; e += 32) {
            const uint32_t k = order_key(to_f32(row[e]));
            if (k) sum += exp((double)key_value<T>(k) - top);
        }
#pragma unroll
        for (int s = 16; s > 0; s /= 2) sum += __shfl_xor_sync(0xffffffffu, sum, s);
    }
    __syncwarp(); // (the groups' 32-bit values lay here)
    for (int e = lane; e < a.experts; e += 32) {
        const uint32_t k = order_key(to_f32(row[e])), b = a.bias ? order_key(a.bias[e]) : 1u;
        double c = none;
        if (k && b) {
            const double l = key_value<T>(k);
            c = a.scoring == SCORING_SIGMOID ? 1.0 / (1.0 + exp(-l)) : exp(l - top) / sum;
            if (a.bias) c += (double)key_value<float>(b);
        }
        values[e] = c;
    }
    __syncwarp();
    const int size = a.experts / a.groups;
    if (a.groups_kept < a.groups) {
        double first = none, second = none; // of group `lane`
        if (lane < a.groups)
            for (int i = 0; i < size; ++i) {
                const double c = values[lane * size + i];
                second = fmax(second, fmin(first, c));
                first = fmax(first, c);
            }
        const double rank = first == none ? none : a.group_best == 2 && second != none ? first + second : first;
        int better = 0;
        for (int g = 0; g < a.groups; ++g) {
            const double other = __shfl_sync(0xffffffffu, rank, g);
            better += other > rank || (other == rank && g < lane);
        }
        if (lane < a.groups && better >= a.groups_kept)
            for (int i = 0; i < size; ++i) values[lane * size + i] = none;
        __syncwarp();
    }
    int mine = -1;
    for (int j = 0; j < a.choices; ++j) {
        double best = none;
        int at = a.experts;
        for (int e = lane; e < a.experts; e += 32)
            if (values[e] > best) {
                best = values[e];
                at = e;
            }
#pragma unroll
        for (int s = 16; s > 0; s /= 2) {
            const double other = __shfl_xor_sync(0xffffffffu, best, s);
            const int other_at = __shfl_xor_sync(0xffffffffu, at, s);
            if (other > best || (other == best && other_at < at)) {
                best = other;
                at = other_at;
            }
        }
        if (best == none) break;
        if (lane == j) mine = at;
        if (at % 32 == lane) values[at] = none;
        __syncwarp();
    }
    return mine;
}

template <typename T, int PER_LANE>
__global__ void __launch_bounds__(WARPS * 32) route_groups_kernel(const __grid_constant__ RouteArgs a) {
    extern __shared__ double shared[];
    ptx::grid_dependency_wait();
    constexpr int V = PER_LANE * sizeof(T) < 16 ? PER_LANE : 16 / (int)sizeof(T); // neighbours that a lane reads at once
    constexpr uint32_t SLOT = PER_LANE - 1; // the bits of a key that say which of the lane's values it is
    const int lane = threadIdx.x & 31;
    const int64_t t = (int64_t)blockIdx.x * WARPS + threadIdx.x / 32;
    if (t >= a.tokens) return;
    const int size = a.experts / a.groups, lanes = group_lanes(a.groups), stride = group_stride(size, lanes);
    double *own = shared + threadIdx.x / 32 * (size_t)((max(2 * a.experts, a.groups_kept < a.groups ? a.groups * stride : 0) + 1) / 2);
    const T *row = (const T *)a.logits + t * a.logits_ld;
    auto expert_of = [&](int i, int l) { return i / V * (32 * V) + l * V + i % V; }; // value i of lane l
    T raw[PER_LANE];
    if (a.aligned) { // rows start on, and hold a multiple of, V values
        struct alignas(V * sizeof(T)) Group { T v[V]; };
#pragma unroll
        for (int i = 0; i < PER_LANE; i += V)
            if (expert_of(i, lane) < a.experts) {
                const Group g = *reinterpret_cast<const Group *>(row + expert_of(i, lane));
#pragma unroll
                for (int j = 0; j < V; ++j) raw[i + j] = g.v[j];
            }
    } else {
#pragma unroll
        for (int i = 0; i < PER_LANE; ++i)
            if (expert_of(i, lane) < a.experts) raw[i] = row[expert_of(i, lane)];
    }
    // scores
    float value[PER_LANE];
    uint32_t there = 0;
    float top = -INFINITY, sum = 0.f;
#pragma unroll
    for (int i = 0; i < PER_LANE; ++i) {
        const float l = to_f32(raw[i]);
        const bool on = expert_of(i, lane) < a.experts && l > -INFINITY; // (not a NaN either)
        there |= on ? 1u << i : 0u;
        value[i] = on ? fminf(l, LARGEST<T>) : -INFINITY;
    }
    if (a.scoring == SCORING_SOFTMAX) {
#pragma unroll
        for (int i = 0; i < PER_LANE; ++i) top = fmaxf(top, value[i]);
        top = warp_max(top);
#pragma unroll
        for (int i = 0; i < PER_LANE; ++i) {
            value[i] = there >> i & 1 ? expf(value[i] - top) : 0.f;
            sum += value[i];
        }
        sum = warp_sum(sum);
        const float inverse = 1.f / sum; // (unused where every expert is masked)
#pragma unroll
        for (int i = 0; i < PER_LANE; ++i) value[i] *= inverse;
    } else {
#pragma unroll
        for (int i = 0; i < PER_LANE; ++i) value[i] = __fdividef(1.f, 1.f + expf(-value[i]));
    }
    float most_bias = 0.f;
    if (a.bias) {
        float bias[PER_LANE];
        if (a.aligned_bias) {
            constexpr int B = V < 4 ? V : 4;
            struct alignas(4 * B) Group { float v[B]; };
#pragma unroll
            for (int i = 0; i < PER_LANE; i += B)
                if (expert_of(i, lane) < a.experts) {
                    const Group g = *reinterpret_cast<const Group *>(a.bias + expert_of(i, lane));
#pragma unroll
                    for (int j = 0; j < B; ++j) bias[i + j] = g.v[j];
                }
        } else {
#pragma unroll
            for (int i = 0; i < PER_LANE; ++i)
                if (expert_of(i, lane) < a.experts) bias[i] = a.bias[expert_of(i, lane)];
        }
#pragma unroll
        for (int i = 0; i < PER_LANE; ++i) {
            const bool on = expert_of(i, lane) < a.experts && bias[i] > -INFINITY;
            if (!on) there &= ~(1u << i);
            const float b = on ? fminf(bias[i], LARGEST<float>) : 0.f;
            most_bias = fmaxf(most_bias, fabsf(b));
            value[i] += b;
        }
        most_bias = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(most_bias)));
    }
    uint32_t key[PER_LANE];
#pragma unroll
    for (int i = 0; i < PER_LANE; ++i) {
        value[i] = there >> i & 1 ? value[i] : -INFINITY;
        key[i] = order_key(value[i]);
    }
    bool close = false; // 32 bits do not tell
    if (a.groups_kept < a.groups) {
        // the two largest of group `lane`
        float first = -INFINITY, second = -INFINITY;
        auto merge = [](float &f, float &s, float f2, float s2) {
            s = fmaxf(fminf(f, f2), fmaxf(s, s2));
            f = fmaxf(f, f2);
        };
        const uint32_t reciprocal = (1u << 20) / size + 1; // e / size for e < 1024: the error stays below 1 / size
        const int span = size / V; // lanes of a group, where a lane's neighbours share one
        if (size % V == 0 && (span & (span - 1)) == 0 && span <= 32) {
            const int per_chunk = 32 / span;
#pragma unroll
            for (int c = 0; c < PER_LANE / V; ++c) {
                float f = -INFINITY, s = -INFINITY;
#pragma unroll
                for (int i = 0; i < V; ++i) merge(f, s, value[c * V + i], -INFINITY);
                for (int d = 1; d < span; d *= 2) merge(f, s, __shfl_xor_sync(0xffffffffu, f, d), __shfl_xor_sync(0xffffffffu, s, d));
                const int from = lane % per_chunk * span;
                const float f2 = __shfl_sync(0xffffffffu, f, from), s2 = __shfl_sync(0xffffffffu, s, from);
                if (lane / per_chunk == c) {
                    first = f2;
                    second = s2;
                }
            }
        } else {
            float *values = (float *)own;
#pragma unroll
            for (int i = 0; i < PER_LANE; ++i) {
                const int e = expert_of(i, lane), g = (int)((e * reciprocal) >> 20);
                if (e < a.experts) values[g * stride + (e - g * size)] = value[i];
            }
            __syncwarp();
            const int group = lane / lanes;
            float f = -INFINITY, s = -INFINITY;
            if (group < a.groups)
                for (int i = lane % lanes; i < size; i += lanes) merge(f, s, values[group * stride + i], -INFINITY);
            for (int d = 1; d < lanes; d *= 2) merge(f, s, __shfl_xor_sync(0xffffffffu, f, d), __shfl_xor_sync(0xffffffffu, s, d));
            first = __shfl_sync(0xffffffffu, f, lane * lanes);
            second = __shfl_sync(0xffffffffu, s, lane * lanes);
        }
        const bool real = lane < a.groups && first > -INFINITY;
        const float rank = !real ? -INFINITY : a.group_best == 2 && second > -INFINITY ? first + second : first;
        int better = 0;
        for (int g = 0; g < a.groups; ++g) {
            const float other = __shfl_sync(0xffffffffu, rank, g);
            better += other > rank || (other == rank && g < lane);
        }
        const uint32_t kept = __ballot_sync(0xffffffffu, real && better < a.groups_kept);
        // the last that is kept and the first that is not: two sums, each of scores up to rank + 2 biases
        const uint32_t ends = __ballot_sync(0xffffffffu, real && better == a.groups_kept - 1), next = __ballot_sync(0xffffffffu, real && better == a.groups_kept);
        if (next) {
            const float l = __shfl_sync(0xffffffffu, rank, __ffs(ends) - 1), n = __shfl_sync(0xffffffffu, rank, __ffs(next) - 1);
            close = !(l - n > 2.f * (score_error(a.scoring) + 0x1p-22f) * (fabsf(l) + 4.f * most_bias));
        }
#pragma unroll
        for (int i = 0; i < PER_LANE; ++i) {
            const int g = (int)((expert_of(i, lane) * reciprocal) >> 20);
            if (!(kept >> (g & 31) & 1)) key[i] = 0;
        }
    }
    uint32_t best = 0;
#pragma unroll
    for (int i = 0; i < PER_LANE; ++i) {
        key[i] = key[i] ? (key[i] & ~SLOT) | (SLOT - i) : 0u;
        best = max(best, key[i]);
    }
    uint32_t mine = 0, owner = 0, several = 0; // lane j: key and lane (as a bit) of choice j
    for (int j = 0; j < a.choices && !close; ++j) {
        const uint32_t most = __reduce_max_sync(0xffffffffu, best);
        if (most == 0) break;
        const uint32_t owners = __ballot_sync(0xffffffffu, best == most);
        if (lane == j) {
            mine = most;
            owner = owners;
        }
        several |= owners & (owners - 1);
        best = next_below(key, most);
    }
    const int slot = (int)(SLOT - (mine & SLOT));
    int index = mine ? expert_of(slot, __ffs(owner) - 1) : -1; // of choice `lane`
    {
        // The next key, of the first that is left out behind the last choice.  Keys differ from c by what the slot's bits hide
        // (2^-23 of the value each), the sum's rounding and the score's error.
        const uint32_t left_out = __reduce_max_sync(0xffffffffu, best), down = __shfl_down_sync(0xffffffffu, mine, 1);
        const uint32_t after = lane == a.choices - 1 ? left_out : down;
        const float c = key_value<float>(mine & ~SLOT), n = key_value<float>(after & ~SLOT);
        const bool near = lane < a.choices && mine && after
                && !(c - n > 2.f * (score_error(a.scoring) + (PER_LANE + 1) * 0x1p-23f) * (fabsf(c) + most_bias));
        close = close || several || __any_sync(0xffffffffu, near);
    }
    if (close) index = choose_in_64_bits(a, row, own);
    const bool chosen = index >= 0;
    const float l = chosen ? key_value<T>(order_key(to_f32(row[index]))) : 0.f;
    float w;
    if (a.scoring == SCORING_SOFTMAX) {
        if (a.normalize) top = warp_max(chosen ? l : -INFINITY);
        w = chosen ? expf(l - top) : 0.f;
        if (a.normalize) sum = warp_sum(w);
        w = chosen ? w / sum : 0.f;
    } else if (a.normalize) {
        const float s = chosen ? log_sigmoid(l) : -INFINITY;
        const float m = warp_max(s);
        w = chosen ? expf(s - m) : 0.f;
        sum = warp_sum(w);
        w = chosen ? w / sum : 0.f;
    } else {
        w = chosen ? sigmoid(l) : 0.f;
    }
    if (lane < a.choices) {
        a.weights[t * a.weights_ld + lane] = w * a.scale;
        a.indices[t * a.indices_ld + lane] = index;
    }
}

template <typename T> int launch_typed(RouteArgs a, cudaStream_t st) {
    const int64_t grid = (a.tokens + WARPS - 1) / WARPS;
    if (grid > 0x7fffffff) return 3;
    const int per_lane = a.experts <= 64 ? 2 : a.experts <= 128 ? 4 : a.experts <= 256 ? 8 : a.experts <= 512 ? 16 : 32;
    const int bytes = std::min(per_lane * (int)sizeof(T), 16), values = bytes / (int)sizeof(T);
    a.aligned = (uintptr_t)a.logits % bytes == 0 && a.experts % values == 0 && (a.tokens == 1 || a.logits_ld % values == 0);
    void (*kernel)(RouteArgs) = per_lane == 2 ? route_groups_kernel<T, 2>
            : per_lane == 4                   ? route_groups_kernel<T, 4>
            : per_lane == 8                   ? route_groups_kernel<T, 8>
            : per_lane == 16                  ? route_groups_kernel<T, 16>
                                              : route_groups_kernel<T, 32>;
    const int grouped = a.groups_kept < a.groups ? a.groups * group_stride(a.experts / a.groups, group_lanes(a.groups)) : 0;
    const size_t smem = (size_t)WARPS * ((std::max(2 * a.experts, grouped) + 1) / 2) * sizeof(double); // at most 40 KB
    const int four = std::min(values, 4);
    a.aligned_bias = a.bias && (uintptr_t)a.bias % (4 * four) == 0 && a.experts % four == 0;
    const int rc = launch_dependent(kernel, a, (unsigned)grid, WARPS * 32, smem, st);
    if (rc == 0) count_launch();
    return rc;
}

} // namespace

int launch_route_groups(const RouteArgs &a, cudaStream_t st) {
    if (a.tokens == 0) return 0;
    switch (a.dt) {
        case DT_F32: return launch_typed<float>(a, st);
        case DT_BF16: return launch_typed<__nv_bfloat16>(a, st);
        case DT_F16: return launch_typed<__half>(a, st);
        default: return 3;
    }
}

} // namespace qmm
