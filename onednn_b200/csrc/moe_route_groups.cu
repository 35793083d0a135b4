// The router's choice by score and bias, within the best groups of experts.
//   score    s = softmax or sigmoid of the logits, as moe_route.cu has them
//   chosen   the k largest of c = s + bias among the experts of the kept groups, which are those whose group_best (1 or 2)
//            largest c have the largest sum; ties go to the lowest group and expert
//   weights  of the chosen, from their scores without the bias
//   masked   logits of -inf and NaN as in moe_route.cu; an expert whose bias is -inf or NaN is never chosen, but counts in a
//            softmax's sum; +inf counts as the largest finite value of its type
// The choice is by the values of c in 64 bits.  32 bits say the same wherever the values that the choice falls between differ by
// more than what rounding can have moved them (8192 x 256: all but some 0.5 % of the rows); only the other rows are
// looked at in 64 bits, out of line: their first candidates, or all experts where the groups are in doubt.  So a warp keeps a row's c
// as 32-bit keys in registers, as moe_route.cu does, with the number of the value in the lane in the lowest bits: keys of a lane differ,
// and a redux and a ballot say which expert it is.  A group's two largest are found in the lanes and by shuffles between them where
// its size allows it, else from shared memory; the groups' ranks by counting.
// Bound by instructions, integer ones above all (8192 x 256 f32, eight groups, k = 8: 16.4 us, floor 1.4; k = 1: 13.0; 2048 rows 7.8;
// one row 4.2).  All of a doubtful row in 64 bits: 19.5, 2048 rows 11.3, one warp's chain of exponentials and code that is in no cache.
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
// And its error besides, where the score is too small for a relative one: a sigmoid below 2^-126 may come out as 0 (its quotient with
// a divisor above 2^126 does), a softmax's is off by a few of the least numbers, 2^-149.  Two scores on either side of a comparison.
constexpr float LEAST_SCORES = 4.f * 0x1p-126f;

// exp(x), x <= 0, in 64 bits without a branch, so that several run at once: x = n log 2 + r with log 2 in two parts of which the
// first has zeros enough that its product with n is exact (Cody and Waite: Software manual for the elementary functions; 1980),
// the series of exp(r) up to r^13 / 13! (what follows is below 2^-57), and n into the exponent; 0 below the least normal number.
__device__ __forceinline__ double exp_64(double x) {
    const double n = rint(x * 1.4426950408889634);
    const double r = fma(-n, 0x1.a39ef35793c76p-33, fma(-n, 0x1.62e42feep-1, x));
    const double r2 = r * r, r4 = r2 * r2;
    const double a = fma(r, 1. / 6, 1. / 2), b = fma(r, 1. / 120, 1. / 24), c = fma(r, 1. / 5040, 1. / 720), d = fma(r, 1. / 362880, 1. / 40320);
    const double e = fma(r, 1. / 39916800, 1. / 3628800), f = fma(r, 1. / 6227020800, 1. / 479001600);
    const double high = fma(r4, fma(r2, f, e), fma(r2, d, c)); // from r^6 on
    const double sum = 1. + (r + r2 * fma(r4, high, fma(r2, b, a)));
    const int k = n > -1023. ? (int)n : -1023;
    return k > -1023 ? sum * __hiloint2double((k + 1023) << 20, 0) : 0.;
}
// 1 / d, 1 <= d <= 2: Newton's steps on the 32-bit reciprocal
__device__ __forceinline__ double inverse_64(double d) {
    double r = __frcp_rn((float)d);
    r = fma(r, fma(-d, r, 1.), r);
    return fma(r, fma(-d, r, 1.), r);
}
// bits in the order of the values, as order_key; 0 for -inf
__device__ __forceinline__ uint64_t order_key_64(double v) {
    const uint64_t u = (uint64_t)__double_as_longlong(v + 0.);
    return v > -INFINITY ? u >> 63 ? ~u : u | 1ull << 63 : 0;
}

// What the 64-bit values of a row are made with: a softmax's largest logit and the inverse of its sum.
struct Row64 { float top; double inverse; };
template <typename T> __device__ __forceinline__ float logit_of(const RouteArgs &a, const T *row, int e, bool &there) {
    const float l = e < a.experts ? to_f32(row[e]) : -INFINITY;
    there = l > -INFINITY;
    return there ? fminf(l, LARGEST<T>) : 0.f;
}
template <typename T> __device__ __forceinline__ Row64 row_in_64_bits(const RouteArgs &a, const T *row) {
    Row64 r {-INFINITY, 1.};
    if (a.scoring == SCORING_SIGMOID) return r;
    const int lane = threadIdx.x & 31;
    bool there;
    for (int e = lane; e < a.experts; e += 32) {
        const float l = logit_of<T>(a, row, e, there);
        if (there) r.top = fmaxf(r.top, l);
    }
    r.top = warp_max(r.top);
    double total = 0;
    for (int e = lane; e < a.experts; e += 32) {
        const float l = logit_of<T>(a, row, e, there);
        const double v = exp_64(there ? (double)l - r.top : 0.);
        total += there ? v : 0.;
    }
#pragma unroll
    for (int s = 16; s > 0; s /= 2) total += __shfl_xor_sync(0xffffffffu, total, s);
    r.inverse = 1. / total; // (unused where every expert is masked)
    return r;
}
// c of an expert, -inf where it cannot be chosen
template <typename T> __device__ __forceinline__ double value_in_64_bits(const RouteArgs &a, const T *row, const Row64 &r, int e) {
    bool there;
    const float l = logit_of<T>(a, row, e, there), b = a.bias && e < a.experts ? a.bias[e] : 0.f;
    const bool sigmoid = a.scoring == SCORING_SIGMOID;
    const double x = exp_64(there ? sigmoid ? -fabs((double)l) : (double)l - r.top : 0.);
    const double scale = sigmoid ? inverse_64(1. + x) : r.inverse;
    const double s = sigmoid && l >= 0.f ? scale : x * scale;
    return there && b > -INFINITY ? s + (double)fminf(b, LARGEST<float>) : -INFINITY;
}

// Lane j of the first `count` has candidate j; returns, in lane j, the one that is j-th by the values in 64 bits, ties to the lowest index.
template <typename T>
__device__ __noinline__ int order_in_64_bits(const RouteArgs &a, const T *row, int candidate, int count) {
    const int lane = threadIdx.x & 31;
    const double c = value_in_64_bits<T>(a, row, row_in_64_bits<T>(a, row), lane < count ? candidate : a.experts);
    int place = 0;
    for (int j = 0; j < count; ++j) {
        const double other = __shfl_sync(0xffffffffu, c, j);
        const int at = __shfl_sync(0xffffffffu, candidate, j);
        place += other > c || (other == c && at < candidate);
    }
    int result = -1;
    for (int j = 0; j < count; ++j) {
        const int to = __shfl_sync(0xffffffffu, place, j), e = __shfl_sync(0xffffffffu, candidate, j);
        if (to == lane) result = e;
    }
    return result;
}

// The k choices of a row in 64 bits.  values: [experts] of this warp's own.  Lane j returns choice j, -1 without one.
template <typename T>
__device__ __noinline__ int choose_in_64_bits(const RouteArgs &a, const T *row, double *values) {
    const int lane = threadIdx.x & 31;
    constexpr double none = -INFINITY;
    const Row64 r = row_in_64_bits<T>(a, row);
    __syncwarp(); // (the groups' 32-bit values lay here)
    for (int e = lane; e < a.experts; e += 32) values[e] = value_in_64_bits<T>(a, row, r, e);
    __syncwarp();
    const int size = a.experts / a.groups, lanes = group_lanes(a.groups);
    if (a.groups_kept < a.groups) {
        double first = none, second = none;
        const int group = lane / lanes;
        if (group < a.groups)
            for (int i = lane % lanes; i < size; i += lanes) {
                const double c = values[group * size + i];
                second = fmax(second, fmin(first, c));
                first = fmax(first, c);
            }
        for (int s = 1; s < lanes; s *= 2) {
            const double f = __shfl_xor_sync(0xffffffffu, first, s), n = __shfl_xor_sync(0xffffffffu, second, s);
            second = fmax(fmin(first, f), fmax(second, n));
            first = fmax(first, f);
        }
        const double rank = first == none ? none : a.group_best == 2 && second != none ? first + second : first;
        int better = 0;
        for (int g = 0; g < a.groups; ++g) {
            const double other = __shfl_sync(0xffffffffu, rank, g * lanes);
            better += other > rank || (other == rank && g < group);
        }
        __syncwarp();
        if (group < a.groups && better >= a.groups_kept)
            for (int i = lane % lanes; i < size; i += lanes) values[group * size + i] = none;
        __syncwarp();
    }
    uint64_t best = 0; // the lane's, and its expert
    int at = 0, mine = -1;
    auto look = [&] {
        best = 0;
        for (int e = lane; e < a.experts; e += 32) {
            const uint64_t k = order_key_64(values[e]);
            if (k > best) {
                best = k;
                at = e;
            }
        }
    };
    look();
    for (int j = 0; j < a.choices; ++j) {
        const uint32_t high = __reduce_max_sync(0xffffffffu, (uint32_t)(best >> 32));
        if (high == 0) break;
        const bool leads = (uint32_t)(best >> 32) == high;
        const uint32_t low = __reduce_max_sync(0xffffffffu, leads ? (uint32_t)best : 0u);
        const int e = __reduce_min_sync(0xffffffffu, leads && (uint32_t)best == low ? at : a.experts);
        if (lane == j) mine = e;
        if (e % 32 == lane) {
            values[e] = none;
            look();
        }
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
        // (two of the lowest biases exceed 32 bits: their group is still in front of those without an expert)
        const float rank = !real ? -INFINITY : a.group_best == 2 && second > -INFINITY ? fmaxf(first + second, -LARGEST<float>) : first;
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
            close = !(l - n > 2.f * (score_error(a.scoring) + 0x1p-22f) * (fabsf(l) + 4.f * most_bias) + LEAST_SCORES);
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
    // Choice after choice; equal keys belong to the same slot of several lanes, and the lowest lane has the lowest expert.
    uint32_t mine = 0; // lane j: key of choice j
    int index = -1; // and its expert
    auto choose = [&](int j) {
        const uint32_t most = __reduce_max_sync(0xffffffffu, best);
        if (most == 0) return false;
        const int owner = __ffs(__ballot_sync(0xffffffffu, best == most)) - 1;
        if (lane == j) {
            mine = most;
            index = owner;
        }
        const uint32_t next = next_below(key, most);
        if (lane == owner) best = next;
        return true;
    };
    int found = 0;
    for (; found < a.choices && !close; ++found)
        if (!choose(found)) break;
    // Whether the next key, of the first that is left out behind the last choice, is so near that 32 bits do not tell.  Keys differ
    // from c by what the slot's bits hide (2^-23 of the value each), the sum's rounding and the score's error.
    uint32_t left_out = __reduce_max_sync(0xffffffffu, best);
    auto near = [&] {
        const uint32_t down = __shfl_down_sync(0xffffffffu, mine, 1), after = lane == found - 1 ? left_out : down;
        const float c = key_value<float>(mine & ~SLOT), n = key_value<float>(after & ~SLOT);
        return lane < found && after && !(c - n > 2.f * (score_error(a.scoring) + (PER_LANE + 1) * 0x1p-23f) * (fabsf(c) + most_bias) + LEAST_SCORES);
    };
    const bool tight = near();
    const bool some = !close && __any_sync(0xffffffffu, tight);
    if (some) { // a few more candidates, up to a gap that 32 bits do tell; in 64 bits their order is found
        while (found < min(a.choices + 4, 32) && choose(found)) ++found;
        left_out = __reduce_max_sync(0xffffffffu, best);
    }
    auto expert_at = [&] { return mine ? expert_of((int)(SLOT - (mine & SLOT)), index) : -1; };
    index = expert_at();
    if (some) {
        const bool gap = !near(); // (by the whole warp)
        const uint32_t gaps = __ballot_sync(0xffffffffu, lane < found && lane >= a.choices - 1 && gap);
        if (found < a.choices) index = order_in_64_bits<T>(a, row, index, found); // (all there are)
        else if (gaps) index = order_in_64_bits<T>(a, row, index, __ffs(gaps));
        else close = true;
    }
    if (close) index = choose_in_64_bits<T>(a, row, own);
    if (lane >= a.choices) index = -1;
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
