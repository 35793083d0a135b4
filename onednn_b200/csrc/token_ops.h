// Plain-data descriptions of one execution of the operators around an expert layer's products (router, sort into grouped
// rows, way back, their gradients) and of dropout, and the entry points that launch their kernels.  Each returns a
// dnnl_status_t value (0 = success, 5 = CUDA runtime error) and only enqueues work on the stream.
#pragma once
#include <cuda_runtime.h>

#include "kernel_args.h"

namespace qmm {

constexpr int TOKEN_MAX_EXPERTS = 1024; // a logit row stays in the registers of a warp; a count per expert in shared memory
constexpr int TOKEN_MAX_CHOICES = 32; // one lane per choice

enum : int { SCORING_SOFTMAX = 0, SCORING_SIGMOID = 1 };

struct RouteArgs {
    int64_t tokens;
    int experts, choices;
    int scoring, normalize;
    float scale;
    int dt; // of the logits and of their gradient
    const void *logits;
    int64_t logits_ld;
    int aligned; // the launcher's: rows can be read several values at a time
    // forward: outputs; backward: indices and the weights' gradient are inputs
    float *weights;
    int64_t weights_ld;
    int *indices;
    int64_t indices_ld;
    void *diff_logits;
    int64_t diff_logits_ld;
};
int launch_route(const RouteArgs &a, cudaStream_t st);
int launch_route_backward(const RouteArgs &a, cudaStream_t st);

struct DispatchArgs {
    int tokens, choices, experts;
    int element; // bytes of one: 1, 2 or 4
    int64_t row_bytes; // of a token's row; the grouped rows are dense
    const char *src;
    int64_t src_pitch; // bytes
    const int *indices;
    int64_t indices_ld;
    char *dst;
    int *offsets; // [experts], cumulative ends
    int *positions;
    int64_t positions_ld;
};
int launch_dispatch(const DispatchArgs &a, int *scratch, int sm_count, cudaStream_t st);
size_t dispatch_scratch_bytes(int experts, int sm_count);

// dropout with a mask that is made again from (seed, offset) wherever it is needed
struct DropoutState {
    const int64_t *seed; // device memory: seed, offset; nullptr: no dropout
    unsigned threshold; // an element is kept where its random word is >= threshold
    int drop_all; // p = 1
    float scale; // 1 / (1 - p)
};

struct CombineArgs {
    int64_t tokens, cols, rows;
    int choices, experts;
    int row_dt, tok_dt; // of the grouped rows; of dst, the residual and diff_dst
    const void *src; // grouped rows, dense
    const int *offsets; // cumulative ends of the groups (the rows behind the last one belong to no slot)
    const int *positions;
    int64_t positions_ld;
    const float *weights; // may be null: 1
    int64_t weights_ld;
    const void *residual; // may be null
    int64_t residual_ld;
    void *dst;
    int64_t dst_ld;
    DropoutState drop;
    int *status; // the engine's status word
    // backward
    const void *diff_dst;
    int64_t diff_dst_ld;
    void *diff_src;
    float *diff_weights;
    int64_t diff_weights_ld;
    unsigned mark_ctas; // the launcher's: CTAs that look for rows without a slot
};
int launch_combine(const CombineArgs &a, int sm_count, cudaStream_t st);
int launch_combine_backward(const CombineArgs &a, int sm_count, cudaStream_t st);

struct DropoutArgs {
    int64_t rows, cols;
    int dt;
    const void *src;
    int64_t src_ld;
    const void *residual; // may be null
    int64_t residual_ld;
    void *dst;
    int64_t dst_ld;
    DropoutState drop;
};
int launch_dropout(const DropoutArgs &a, int sm_count, cudaStream_t st);

// Launches `kernel` as a programmatic dependent of whatever precedes it on the stream; the kernel reads and writes global
// memory behind griddepcontrol.wait only.
template <typename Args>
inline int launch_dependent(void (*kernel)(Args), const Args &a, unsigned grid, unsigned block, size_t smem, cudaStream_t st) {
    cudaLaunchConfig_t cfg {};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(block);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    void *kargs[] = {const_cast<Args *>(&a)};
    return cudaLaunchKernelExC(&cfg, (const void *)kernel, kargs) == cudaSuccess ? 0 : 5;
}

} // namespace qmm
