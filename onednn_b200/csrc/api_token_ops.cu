// Descriptors and execution of the operators around an expert layer's products, of dropout, of the norm and of low-rank adapters (dnnl_b200.h).  One check
// serves creation and, where dims were left open, each execution: it skips what an open dim leaves unsaid.
#include <initializer_list>
#include <memory>
#include <new>

#include "launch.h"
#include "objects.hpp"
#include "token_ops.h"

using namespace qmm;

namespace {

constexpr dnnl_dim_t OPEN = DNNL_RUNTIME_DIM_VAL;
constexpr dnnl_dim_t MAX_SLOTS = (dnnl_dim_t)1 << 30;

bool agree(dnnl_dim_t a, dnnl_dim_t b) { return a == OPEN || b == OPEN || a == b; }

bool is_float(int dt) { return dt == dnnl_f32 || dt == dnnl_bf16 || dt == dnnl_f16; }

struct checker_t {
    dnnl_status_t status = dnnl_success;
    void fail(dnnl_status_t s) {
        // an argument error outranks what is merely not built
        if (status == dnnl_success || (status == dnnl_unimplemented && s == dnnl_invalid_arguments)) status = s;
    }
    void require(bool ok) { if (!ok) fail(dnnl_invalid_arguments); }
    void built(bool ok) { if (!ok) fail(dnnl_unimplemented); }
    // a matrix with neighbouring columns beside one another
    bool matrix(const dnnl_memory_desc *md, bool output) {
        require(md && md->ndims == 2 && md->format_kind != dnnl_format_kind_undef);
        if (!md || md->ndims != 2 || md->format_kind == dnnl_format_kind_undef) return false;
        built(md->format_kind == dnnl_blocked);
        if (md->format_kind != dnnl_blocked) return false;
        if (md->dims[0] == 0 || md->dims[1] == 0) return true; // (nothing is read: any strides)
        built(md->dims[1] == 1 || md->strides[1] == 1 || md->strides[1] == OPEN);
        const bool known = md->dims[0] != OPEN && md->dims[1] != OPEN && md->strides[0] != OPEN;
        if (output && known && md->dims[0] > 1) built(md->strides[0] >= md->dims[1]);
        return true;
    }
    // [rows, cols] of one of the given types
    bool matrix(const dnnl_memory_desc *md, bool output, dnnl_dim_t rows, dnnl_dim_t cols, dnnl_data_type_t dt) {
        if (!matrix(md, output)) return false;
        require(agree(md->dims[0], rows) && agree(md->dims[1], cols));
        built(md->data_type == dt);
        return true;
    }
    // `n` neighbouring values
    bool vector(const dnnl_memory_desc *md, dnnl_dim_t n) {
        require(md && md->ndims == 1 && md->format_kind != dnnl_format_kind_undef);
        if (!md || md->ndims != 1 || md->format_kind == dnnl_format_kind_undef) return false;
        built(md->format_kind == dnnl_blocked);
        if (md->format_kind != dnnl_blocked) return false;
        require(agree(md->dims[0], n));
        built(md->dims[0] == 0 || md->dims[0] == 1 || md->strides[0] == 1);
        return true;
    }
    // [a, b, c], strided anyhow
    bool cube(const dnnl_memory_desc *md, dnnl_dim_t a, dnnl_dim_t b, dnnl_dim_t c) {
        require(md && md->ndims == 3 && md->format_kind != dnnl_format_kind_undef);
        if (!md || md->ndims != 3 || md->format_kind == dnnl_format_kind_undef) return false;
        built(md->format_kind == dnnl_blocked);
        require(agree(md->dims[0], a) && agree(md->dims[1], b) && agree(md->dims[2], c));
        return md->format_kind == dnnl_blocked;
    }
    bool grouped(const dnnl_memory_desc *md, dnnl_dim_t rows, dnnl_dim_t cols, dnnl_dim_t groups) {
        require(md && md->is_grouped());
        if (!md || !md->is_grouped()) return false;
        require(md->ndims == 2 && md->variable_dim_idx == 0 && agree(md->dims[0], rows) && agree(md->dims[1], cols)
                && (groups == 0 || md->group_count == groups));
        built(md->group_count <= TOKEN_MAX_EXPERTS);
        return true;
    }
    void choices(dnnl_dim_t tokens, dnnl_dim_t k) {
        if (k == OPEN) return;
        require(k >= 1);
        built(k <= TOKEN_MAX_CHOICES);
        if (tokens != OPEN && k >= 1) built(tokens <= MAX_SLOTS / k);
    }
};

dnnl_dim_t known(dnnl_dim_t a, dnnl_dim_t b) { return a == OPEN ? b : a; }
dnnl_dim_t times(dnnl_dim_t a, dnnl_dim_t b) { return a == OPEN || b == OPEN || a > MAX_SLOTS || b > MAX_SLOTS ? OPEN : a * b; }

// src, weights and sizes of the norm and of its gradient
void norm_common(checker_t &c, const token_op_t &op, const dnnl_memory_desc *src, dnnl_dim_t T, dnnl_dim_t H, const dnnl_memory_desc *wei) {
    c.require(op.epsilon > 0.f && op.epsilon - op.epsilon == 0.f);
    c.built(is_float(src->data_type));
    if (wei && c.vector(wei, H)) c.built(wei->data_type == dnnl_f32 || wei->data_type == src->data_type);
    if (H != OPEN) {
        c.require(H >= 1);
        c.built(H <= NORM_MAX_COLS);
    }
    if (T != OPEN) c.built(T <= MAX_SLOTS);
}

// the tensor whose scales an attribute may set
int scaled_arg(int kind) {
    return kind == dnnl_cuda_interop_rms_norm ? DNNL_ARG_DST : kind == dnnl_cuda_interop_low_rank_adapter ? DNNL_ARG_WEIGHTS : 0;
}

// the tensor's dims that the mask names, divided by the groups, dense
dnnl_memory_desc scales_md(const quant_entry_t &q, const dnnl_memory_desc &base) {
    dnnl_memory_desc md;
    md.ndims = base.ndims;
    md.data_type = q.dt;
    md.format_kind = dnnl_blocked;
    dnnl_dim_t stride = 1;
    for (int i = base.ndims - 1; i >= 0; --i) {
        const dnnl_dim_t g = q.group_ndims && i >= base.ndims - 2 ? q.groups[i - (base.ndims - 2)] : 1;
        md.dims[i] = !((q.mask >> i) & 1) ? 1 : base.dims[i] == OPEN ? OPEN : base.dims[i] / g;
        md.strides[i] = stride;
        stride = stride == OPEN || md.dims[i] == OPEN ? OPEN : stride * md.dims[i];
    }
    return md;
}

dnnl_status_t check(int kind, const token_op_t &op) {
    checker_t c;
    const auto *src = op.find(DNNL_ARG_SRC), *src1 = op.find(DNNL_ARG_SRC_1), *src2 = op.find(DNNL_ARG_SRC_2);
    const auto *wei = op.find(DNNL_ARG_WEIGHTS), *dst = op.find(DNNL_ARG_DST), *dst1 = op.find(DNNL_ARG_DST_1);
    const auto *dsrc = op.find(DNNL_ARG_DIFF_SRC), *ddst = op.find(DNNL_ARG_DIFF_DST), *dwei = op.find(DNNL_ARG_DIFF_WEIGHTS);
    c.require(op.p >= 0.f && op.p <= 1.f); // (not a NaN either)
    switch (kind) {
        case dnnl_cuda_interop_moe_route:
        case dnnl_cuda_interop_moe_route_backward: {
            const bool backward = kind == dnnl_cuda_interop_moe_route_backward;
            c.require(op.scoring == SCORING_SOFTMAX || op.scoring == SCORING_SIGMOID);
            c.require(op.scale - op.scale == 0.f); // finite
            const auto *indices = backward ? src1 : dst1, *weights = backward ? ddst : dst;
            if (!c.matrix(src, false) || !c.matrix(indices, !backward) || !c.matrix(weights, !backward)) break;
            const dnnl_dim_t T = known(src->dims[0], indices->dims[0]), E = src->dims[1];
            const dnnl_dim_t K = known(indices->dims[1], weights->dims[1]);
            c.matrix(indices, !backward, T, K, dnnl_s32);
            c.matrix(weights, !backward, T, K, dnnl_f32);
            c.require(agree(src->dims[0], weights->dims[0]));
            c.built(is_float(src->data_type));
            if (E != OPEN) {
                c.require(E >= 1 && (K == OPEN || K <= E));
                c.built(E <= TOKEN_MAX_EXPERTS);
            }
            c.choices(T, K);
            if (const auto *bias = op.find(DNNL_ARG_BIAS))
                if (c.vector(bias, E)) c.built(bias->data_type == dnnl_f32);
            c.require(op.groups >= 1 && op.groups_kept >= 1 && op.groups_kept <= op.groups && (op.group_best == 1 || op.group_best == 2));
            c.built(op.groups <= TOKEN_MAX_GROUPS);
            if (E != OPEN && op.groups >= 1) {
                c.require(E % op.groups == 0);
                if (K != OPEN) c.require(K <= E / op.groups * op.groups_kept);
            }
            if (backward) c.matrix(dsrc, true, T, E, src->data_type);
            break;
        }
        case dnnl_cuda_interop_moe_dispatch: {
            if (!c.matrix(src, false) || !c.matrix(src1, false) || !c.matrix(dst1, true)) break;
            const dnnl_dim_t T = known(src->dims[0], src1->dims[0]), K = known(src1->dims[1], dst1->dims[1]);
            c.matrix(src1, false, T, K, dnnl_s32);
            c.matrix(dst1, true, T, K, dnnl_s32);
            c.choices(T, K);
            if (!c.grouped(dst, times(T, K), src->dims[1], 0)) break;
            const size_t bits = dt_bits(src->data_type);
            c.built(bits == 8 || bits == 16 || bits == 32);
            c.require(dst->data_type == src->data_type);
            break;
        }
        case dnnl_cuda_interop_moe_combine: {
            if (!c.matrix(dst, true) || !c.matrix(src1, false)) break;
            const dnnl_dim_t T = known(dst->dims[0], src1->dims[0]), K = src1->dims[1], H = dst->dims[1];
            c.matrix(src1, false, T, K, dnnl_s32);
            c.choices(T, K);
            if (wei) c.matrix(wei, false, T, K, dnnl_f32);
            if (src2) c.matrix(src2, false, T, H, dst->data_type);
            if (!c.grouped(src, times(T, K), H, 0)) break;
            c.built(is_float(src->data_type) && is_float(dst->data_type));
            break;
        }
        case dnnl_cuda_interop_moe_combine_backward: {
            if (!c.matrix(ddst, false) || !c.matrix(src1, false)) break;
            const dnnl_dim_t T = known(ddst->dims[0], src1->dims[0]), K = src1->dims[1], H = ddst->dims[1];
            c.matrix(src1, false, T, K, dnnl_s32);
            c.choices(T, K);
            c.matrix(wei, false, T, K, dnnl_f32);
            c.matrix(dwei, true, T, K, dnnl_f32);
            if (!c.grouped(src, times(T, K), H, 0)) break;
            if (!c.grouped(dsrc, times(T, K), H, src->group_count)) break;
            c.built(is_float(src->data_type) && is_float(ddst->data_type) && dsrc->data_type == src->data_type);
            break;
        }
        case dnnl_cuda_interop_dropout: {
            if (!c.matrix(src, false) || !c.matrix(dst, true)) break;
            c.matrix(dst, true, src->dims[0], src->dims[1], src->data_type);
            if (src2) c.matrix(src2, false, src->dims[0], src->dims[1], src->data_type);
            c.built(is_float(src->data_type));
            break;
        }
        case dnnl_cuda_interop_rms_norm: {
            if (!c.matrix(src, false) || !c.matrix(dst, true)) break;
            const dnnl_dim_t T = known(src->dims[0], dst->dims[0]), H = known(src->dims[1], dst->dims[1]);
            c.matrix(src, false, T, H, src->data_type);
            c.matrix(dst, true, T, H, dst->data_type);
            norm_common(c, op, src, T, H, wei);
            if (src2) c.matrix(src2, false, T, H, src->data_type);
            if (dst1) c.matrix(dst1, true, T, H, src->data_type);
            const bool small = dst->data_type == dnnl_s8 || dst->data_type == dnnl_f8_e4m3;
            c.built(small || dst->data_type == dnnl_f32 || dst->data_type == src->data_type);
            if (op.scaling != NORM_SCALE_NONE) c.built(small);
            if (op.scaling == NORM_SCALE_GROUP && H != OPEN) c.require(H % op.group == 0);
            break;
        }
        case dnnl_cuda_interop_rms_norm_backward: {
            if (!c.matrix(ddst, false) || !c.matrix(src, false) || !c.matrix(dsrc, true)) break;
            const dnnl_dim_t T = known(known(ddst->dims[0], src->dims[0]), dsrc->dims[0]);
            const dnnl_dim_t H = known(known(ddst->dims[1], src->dims[1]), dsrc->dims[1]);
            c.matrix(src, false, T, H, src->data_type);
            c.matrix(ddst, false, T, H, src->data_type);
            c.matrix(dsrc, true, T, H, src->data_type);
            norm_common(c, op, src, T, H, wei);
            if (src2) c.matrix(src2, false, T, H, src->data_type);
            if (dwei && c.vector(dwei, H)) {
                c.built(H != OPEN); // (its scratchpad is made before the first execution)
                c.built(dwei->data_type == dnnl_f32 || dwei->data_type == src->data_type);
            }
            break;
        }
        case dnnl_cuda_interop_low_rank_adapter: {
            const auto *up = op.find(DNNL_ARG_WEIGHTS_1);
            if (!c.matrix(src, false) || !c.matrix(dst, true) || !c.cube(wei, OPEN, OPEN, OPEN) || !c.cube(up, OPEN, OPEN, OPEN)) break;
            if (!c.vector(src1, OPEN)) break;
            const dnnl_dim_t T = known(known(src->dims[0], dst->dims[0]), src1->dims[0]), n = known(wei->dims[0], up->dims[0]);
            const dnnl_dim_t r = known(wei->dims[2], up->dims[1]);
            c.require(agree(src->dims[0], T) && agree(dst->dims[0], T) && agree(src1->dims[0], T));
            c.cube(wei, n, src->dims[1], r);
            c.cube(up, n, r, dst->dims[1]);
            if (src2) c.matrix(src2, false, T, dst->dims[1], dst->data_type);
            c.built(src1->data_type == dnnl_s32 && (src->data_type == dnnl_bf16 || src->data_type == dnnl_f16));
            c.built(wei->data_type == src->data_type && up->data_type == src->data_type);
            c.built(dst->data_type == src->data_type || dst->data_type == dnnl_f32);
            if (n != OPEN) {
                c.require(n >= 1);
                c.built(n <= LOW_RANK_MAX_ADAPTERS);
            }
            if (r != OPEN) {
                c.require(r >= 1);
                c.built(r <= LOW_RANK_MAX);
            }
            for (dnnl_dim_t d : {T, src->dims[1], dst->dims[1]})
                if (d != OPEN) c.built(d <= MAX_SLOTS);
            break;
        }
        default: return dnnl_invalid_arguments;
    }
    return c.status;
}

// Scales that an attribute asks for: how they are made or given, and their descriptor among the tensors.
dnnl_status_t add_scales(int kind, token_op_t &op, const dnnl_primitive_attr &attr) {
    const int arg = scaled_arg(kind);
    const quant_entry_t &q = attr.scale(arg);
    if (!arg || !q.set) return dnnl_success;
    if (q.dt != dnnl_f32 || q.on_host) return dnnl_unimplemented;
    if (kind == dnnl_cuda_interop_rms_norm) {
        const bool made = q.qmode == dnnl_quantization_mode_dynamic_fp;
        if (q.mask == 0 && q.qmode == dnnl_quantization_mode_static_sazp) op.scaling = NORM_SCALE_GIVEN;
        else if (q.mask == 1 && made && !q.group_ndims) op.scaling = NORM_SCALE_ROW;
        else if (q.mask == 3 && made && q.group_ndims && q.groups[0] == 1) {
            const dnnl_dim_t g = q.groups[1];
            if (g < 16 || g > 256 || (g & (g - 1))) return dnnl_unimplemented;
            op.scaling = NORM_SCALE_GROUP;
            op.group = (int)g;
        } else return dnnl_unimplemented;
    } else if (q.mask != 1 || q.group_ndims || q.qmode != dnnl_quantization_mode_static_sazp) { // one per adapter
        return dnnl_unimplemented;
    }
    op.args[DNNL_ARG_ATTR_SCALES | arg] = scales_md(q, *op.find(arg));
    return dnnl_success;
}

// A null or zero descriptor leaves an optional tensor out, and is an error for the others.
dnnl_status_t create(dnnl_primitive_desc_t *out, dnnl_engine_t engine, int kind, token_op_t op,
        std::initializer_list<std::pair<int, const_dnnl_memory_desc_t>> tensors,
        std::initializer_list<std::pair<int, const_dnnl_memory_desc_t>> optional, const_dnnl_primitive_attr_t attr) try {
    if (!out || !engine) return dnnl_invalid_arguments;
    for (const auto &t : tensors) {
        if (!t.second) return dnnl_invalid_arguments;
        op.args[t.first] = *t.second;
    }
    for (const auto &t : optional)
        if (t.second && !t.second->is_zero()) op.args[t.first] = *t.second;
    dnnl_status_t st = check(kind, op);
    if (st != dnnl_success) return st;
    if (attr) {
        dnnl_primitive_attr plain = *attr;
        plain.scratchpad_mode = dnnl_scratchpad_mode_library;
        if (scaled_arg(kind)) plain.scales.erase(scaled_arg(kind));
        if (!plain.has_default_values()) return dnnl_unimplemented;
        st = add_scales(kind, op, *attr);
        if (st == dnnl_success && op.scaling != NORM_SCALE_NONE) st = check(kind, op);
        if (st != dnnl_success) return st;
    }
    if (op.p > 0.f || kind == dnnl_cuda_interop_dropout) { // (seed, offset)
        dnnl_memory_desc seed;
        seed.ndims = 1;
        seed.dims[0] = 2;
        seed.strides[0] = 1;
        seed.data_type = dnnl_s64;
        seed.format_kind = dnnl_blocked;
        op.args[DNNL_ARG_ATTR_DROPOUT_SEED] = seed;
    }
    std::unique_ptr<dnnl_primitive_desc> pd(new dnnl_primitive_desc);
    pd->kind = kind;
    pd->engine = engine;
    if (attr) pd->attr = *attr;
    pd->impl_name = std::string("cuda:simt:") + token_op_name(kind);
    if (kind == dnnl_cuda_interop_moe_dispatch)
        pd->scratch_bytes = dispatch_scratch_bytes((int)op.args[DNNL_ARG_DST].group_count, engine->sm_count > 0 ? engine->sm_count : 148);
    if (kind == dnnl_cuda_interop_rms_norm_backward && op.find(DNNL_ARG_DIFF_WEIGHTS)) {
        const dnnl_dim_t cols[] = {op.find(DNNL_ARG_DIFF_WEIGHTS)->dims[0], op.find(DNNL_ARG_SRC)->dims[1],
                op.find(DNNL_ARG_DIFF_DST)->dims[1], op.find(DNNL_ARG_DIFF_SRC)->dims[1]};
        dnnl_dim_t known_cols = OPEN;
        for (dnnl_dim_t n : cols) known_cols = known(known_cols, n);
        pd->scratch_bytes = norm_scratch_bytes(known_cols, engine->sm_count > 0 ? engine->sm_count : 148);
    }
    if (kind == dnnl_cuda_interop_low_rank_adapter) {
        const dnnl_dim_t rows = known(known(op.find(DNNL_ARG_SRC)->dims[0], op.find(DNNL_ARG_DST)->dims[0]), op.find(DNNL_ARG_SRC_1)->dims[0]);
        const dnnl_dim_t rank = known(op.find(DNNL_ARG_WEIGHTS)->dims[2], op.find(DNNL_ARG_WEIGHTS_1)->dims[1]);
        pd->scratch_bytes = low_rank_scratch_bytes(rows, rank);
    }
    if (pd->scratch_bytes && pd->attr.scratchpad_mode == dnnl_scratchpad_mode_user) {
        pd->scratchpad.ndims = 1;
        pd->scratchpad.dims[0] = (dnnl_dim_t)pd->scratch_bytes;
        pd->scratchpad.strides[0] = 1;
        pd->scratchpad.data_type = dnnl_u8;
        pd->scratchpad.format_kind = dnnl_blocked;
    }
    pd->token_op = std::move(op);
    *out = pd.release();
    return dnnl_success;
} catch (const std::bad_alloc &) { // no exception leaves a C entry
    return dnnl_out_of_memory;
}

// where an execution's tensors are
struct bound_t {
    struct { int arg; char *values; const int *offsets; } t[10];
    int n = 0;
};

int launch(const dnnl_primitive &primitive, int kind, const token_op_t &op, const bound_t &bound, void *scratch, cudaStream_t stream) {
    const int sms = primitive.pd.engine->sm_count > 0 ? primitive.pd.engine->sm_count : 148;
    auto ptr = [&](int arg) -> void * {
        for (int i = 0; i < bound.n; ++i)
            if (bound.t[i].arg == arg) return bound.t[i].values;
        return nullptr;
    };
    auto ends = [&](int arg) -> const int * {
        for (int i = 0; i < bound.n; ++i)
            if (bound.t[i].arg == arg) return bound.t[i].offsets;
        return nullptr;
    };
    // row pitch in elements (of a single row: its width)
    auto ld = [&](int arg) -> int64_t {
        const auto *md = op.find(arg);
        return !md ? 0 : md->dims[0] > 1 ? md->strides[0] : md->dims[1];
    };
    DropoutState drop {};
    if (op.find(DNNL_ARG_ATTR_DROPOUT_SEED)) {
        drop.seed = (const int64_t *)ptr(DNNL_ARG_ATTR_DROPOUT_SEED);
        drop.drop_all = op.p >= 1.f;
        drop.threshold = drop.drop_all ? 0xffffffffu : (unsigned)((double)op.p * 4294967296.0);
        drop.scale = drop.drop_all ? 0.f : (float)(1.0 / (1.0 - (double)op.p));
    }
    switch (kind) {
        case dnnl_cuda_interop_moe_route:
        case dnnl_cuda_interop_moe_route_backward: {
            const bool backward = kind == dnnl_cuda_interop_moe_route_backward;
            const int weights = backward ? DNNL_ARG_DIFF_DST : DNNL_ARG_DST, indices = backward ? DNNL_ARG_SRC_1 : DNNL_ARG_DST_1;
            const auto *src = op.find(DNNL_ARG_SRC);
            RouteArgs a {};
            a.tokens = src->dims[0]; a.experts = (int)src->dims[1]; a.choices = (int)op.find(indices)->dims[1];
            a.scoring = op.scoring; a.normalize = op.normalize; a.scale = op.scale;
            a.dt = src->data_type;
            a.logits = ptr(DNNL_ARG_SRC); a.logits_ld = ld(DNNL_ARG_SRC);
            a.weights = (float *)ptr(weights); a.weights_ld = ld(weights);
            a.indices = (int *)ptr(indices); a.indices_ld = ld(indices);
            a.bias = (const float *)ptr(DNNL_ARG_BIAS);
            a.groups = op.groups; a.groups_kept = op.groups_kept; a.group_best = op.group_best;
            a.diff_logits = ptr(DNNL_ARG_DIFF_SRC); a.diff_logits_ld = ld(DNNL_ARG_DIFF_SRC);
            return backward ? launch_route_backward(a, stream) : launch_route(a, stream);
        }
        case dnnl_cuda_interop_moe_dispatch: {
            const auto *src = op.find(DNNL_ARG_SRC);
            const int64_t size = (int64_t)dt_bits(src->data_type) / 8;
            DispatchArgs a {};
            a.tokens = (int)src->dims[0]; a.choices = (int)op.find(DNNL_ARG_SRC_1)->dims[1];
            a.experts = (int)op.find(DNNL_ARG_DST)->group_count;
            a.element = (int)size;
            a.row_bytes = src->dims[1] * size;
            a.src = (const char *)ptr(DNNL_ARG_SRC); a.src_pitch = ld(DNNL_ARG_SRC) * size;
            a.indices = (const int *)ptr(DNNL_ARG_SRC_1); a.indices_ld = ld(DNNL_ARG_SRC_1);
            a.dst = (char *)ptr(DNNL_ARG_DST);
            a.offsets = const_cast<int *>(ends(DNNL_ARG_DST));
            a.positions = (int *)ptr(DNNL_ARG_DST_1); a.positions_ld = ld(DNNL_ARG_DST_1);
            return launch_dispatch(a, (int *)scratch, sms, stream);
        }
        case dnnl_cuda_interop_moe_combine:
        case dnnl_cuda_interop_moe_combine_backward: {
            const bool backward = kind == dnnl_cuda_interop_moe_combine_backward;
            const int tokens = backward ? DNNL_ARG_DIFF_DST : DNNL_ARG_DST;
            const auto *tok = op.find(tokens), *rows = op.find(DNNL_ARG_SRC);
            CombineArgs a {};
            a.tokens = tok->dims[0]; a.cols = tok->dims[1]; a.rows = rows->dims[0];
            a.choices = (int)op.find(DNNL_ARG_SRC_1)->dims[1]; a.experts = (int)rows->group_count;
            a.row_dt = rows->data_type; a.tok_dt = tok->data_type;
            a.src = ptr(DNNL_ARG_SRC); a.offsets = ends(DNNL_ARG_SRC);
            a.positions = (const int *)ptr(DNNL_ARG_SRC_1); a.positions_ld = ld(DNNL_ARG_SRC_1);
            a.weights = (const float *)ptr(DNNL_ARG_WEIGHTS); a.weights_ld = ld(DNNL_ARG_WEIGHTS);
            a.residual = ptr(DNNL_ARG_SRC_2); a.residual_ld = ld(DNNL_ARG_SRC_2);
            a.dst = ptr(DNNL_ARG_DST); a.dst_ld = ld(DNNL_ARG_DST);
            a.drop = drop;
            a.status = primitive.pd.engine->status_word;
            a.diff_dst = ptr(DNNL_ARG_DIFF_DST); a.diff_dst_ld = ld(DNNL_ARG_DIFF_DST);
            a.diff_src = ptr(DNNL_ARG_DIFF_SRC);
            a.diff_weights = (float *)ptr(DNNL_ARG_DIFF_WEIGHTS); a.diff_weights_ld = ld(DNNL_ARG_DIFF_WEIGHTS);
            return backward ? launch_combine_backward(a, sms, stream) : launch_combine(a, sms, stream);
        }
        case dnnl_cuda_interop_rms_norm:
        case dnnl_cuda_interop_rms_norm_backward: {
            const bool backward = kind == dnnl_cuda_interop_rms_norm_backward;
            const auto *src = op.find(DNNL_ARG_SRC), *dst = op.find(DNNL_ARG_DST), *wei = op.find(DNNL_ARG_WEIGHTS);
            const auto *dwei = op.find(DNNL_ARG_DIFF_WEIGHTS);
            NormArgs a {};
            a.rows = src->dims[0]; a.cols = src->dims[1]; a.dt = src->data_type;
            a.src = ptr(DNNL_ARG_SRC); a.src_ld = ld(DNNL_ARG_SRC);
            a.residual = ptr(DNNL_ARG_SRC_2); a.residual_ld = ld(DNNL_ARG_SRC_2);
            a.epsilon = op.epsilon;
            a.weights = ptr(DNNL_ARG_WEIGHTS); a.weights_dt = wei ? wei->data_type : dnnl_f32;
            if (backward) {
                a.diff_dst = ptr(DNNL_ARG_DIFF_DST); a.diff_dst_ld = ld(DNNL_ARG_DIFF_DST);
                a.diff_src = ptr(DNNL_ARG_DIFF_SRC); a.diff_src_ld = ld(DNNL_ARG_DIFF_SRC);
                a.diff_weights = ptr(DNNL_ARG_DIFF_WEIGHTS); a.weights_grad_dt = dwei ? dwei->data_type : dnnl_f32;
                a.parts = a.diff_weights ? (float *)scratch : nullptr;
                return launch_rms_norm_backward(a, sms, stream);
            }
            a.sum = ptr(DNNL_ARG_DST_1); a.sum_ld = ld(DNNL_ARG_DST_1);
            a.dst = ptr(DNNL_ARG_DST); a.dst_ld = ld(DNNL_ARG_DST); a.dst_dt = dst->data_type;
            a.scaling = op.scaling; a.group = op.group;
            a.scales = (float *)ptr(DNNL_ARG_ATTR_SCALES | DNNL_ARG_DST);
            return launch_rms_norm(a, sms, stream);
        }
        case dnnl_cuda_interop_low_rank_adapter: {
            const auto *src = op.find(DNNL_ARG_SRC), *dst = op.find(DNNL_ARG_DST), *down = op.find(DNNL_ARG_WEIGHTS), *up = op.find(DNNL_ARG_WEIGHTS_1);
            LowRankArgs a {};
            a.rows = src->dims[0]; a.in = src->dims[1]; a.out = dst->dims[1];
            a.adapters = (int)down->dims[0]; a.rank = (int)down->dims[2];
            a.dt = src->data_type; a.dst_dt = dst->data_type;
            a.src = ptr(DNNL_ARG_SRC); a.src_ld = ld(DNNL_ARG_SRC);
            a.indices = (const int *)ptr(DNNL_ARG_SRC_1);
            a.down = ptr(DNNL_ARG_WEIGHTS); a.down_adapter = down->strides[0]; a.down_in = down->strides[1]; a.down_rank = down->strides[2];
            a.up = ptr(DNNL_ARG_WEIGHTS_1); a.up_adapter = up->strides[0]; a.up_rank = up->strides[1]; a.up_out = up->strides[2];
            a.scales = (const float *)ptr(DNNL_ARG_ATTR_SCALES | DNNL_ARG_WEIGHTS);
            a.base = ptr(DNNL_ARG_SRC_2); a.base_ld = ld(DNNL_ARG_SRC_2);
            a.dst = ptr(DNNL_ARG_DST); a.dst_ld = ld(DNNL_ARG_DST);
            return launch_low_rank(a, scratch, sms, stream);
        }
        default: {
            const auto *src = op.find(DNNL_ARG_SRC);
            DropoutArgs a {};
            a.rows = src->dims[0]; a.cols = src->dims[1]; a.dt = src->data_type;
            a.src = ptr(DNNL_ARG_SRC); a.src_ld = ld(DNNL_ARG_SRC);
            a.residual = ptr(DNNL_ARG_SRC_2); a.residual_ld = ld(DNNL_ARG_SRC_2);
            a.dst = ptr(DNNL_ARG_DST); a.dst_ld = ld(DNNL_ARG_DST);
            a.drop = drop;
            return launch_dropout(a, sms, stream);
        }
    }
}

} // namespace

namespace qmm {

bool is_token_op(int kind) {
    return (kind >= dnnl_cuda_interop_moe_route && kind <= dnnl_cuda_interop_dropout)
            || (kind >= dnnl_cuda_interop_rms_norm && kind <= dnnl_cuda_interop_low_rank_adapter);
}

const char *token_op_name(int kind) {
    static const char *const names[] = {"moe_route", "moe_route_backward", "moe_dispatch", "moe_combine", "moe_combine_backward", "dropout"};
    static const char *const later[] = {"rms_norm", "rms_norm_backward", "low_rank_adapter"};
    if (!is_token_op(kind)) return "unknown";
    return kind >= dnnl_cuda_interop_rms_norm ? later[kind - dnnl_cuda_interop_rms_norm] : names[kind - dnnl_cuda_interop_moe_route];
}

dnnl_status_t execute_token_op(const dnnl_primitive &primitive, dnnl_stream_t stream, int nargs, const dnnl_exec_arg_t *args) try {
    const dnnl_primitive_desc &pd = primitive.pd;
    auto find = [&](int key) -> dnnl_memory_t {
        for (int i = 0; i < nargs; ++i)
            if (args[i].arg == key) return args[i].memory;
        return nullptr;
    };
    bool open = false;
    for (const auto &kv : pd.token_op.args) {
        open = open || kv.second.has_runtime_dims();
        if (!find(kv.first)) return dnnl_invalid_arguments;
    }
    for (int i = 0; i < nargs; ++i) // a tensor the descriptor does not know would be ignored in silence
        if (args[i].arg != DNNL_ARG_SCRATCHPAD && !pd.token_op.find(args[i].arg)) return dnnl_invalid_arguments;
    // dims left open: every descriptor from its memory object, which must agree with what was stated
    token_op_t settled;
    const token_op_t *op = &pd.token_op;
    if (open) {
        settled = pd.token_op;
        for (auto &kv : settled.args) {
            dnnl_memory_desc &want = kv.second;
            if (kv.first == DNNL_ARG_ATTR_DROPOUT_SEED || (kv.first & DNNL_ARG_ATTR_SCALES)) continue;
            const dnnl_memory_desc &got = find(kv.first)->md;
            if (got.ndims != want.ndims || got.has_runtime_dims() || got.data_type != want.data_type
                    || got.format_kind != want.format_kind || got.is_grouped() != want.is_grouped()
                    || got.group_count != want.group_count)
                return dnnl_invalid_arguments;
            for (int d = 0; d < want.ndims; ++d)
                if (!agree(want.dims[d], got.dims[d])) return dnnl_invalid_arguments;
            want = got;
        }
        const dnnl_status_t st = check(pd.kind, settled);
        if (st != dnnl_success) return st;
        const int scaled = scaled_arg(pd.kind), scales = DNNL_ARG_ATTR_SCALES | scaled;
        if (settled.find(scales)) { // made from the settled tensor; the memory object has to hold as many
            settled.args[scales] = scales_md(pd.attr.scale(scaled), *settled.find(scaled));
            const dnnl_memory_desc &got = find(scales)->md;
            if (got.data_type != dnnl_f32 || got.format_kind != dnnl_blocked || got.has_runtime_dims()
                    || got.nelems() < settled.find(scales)->nelems())
                return dnnl_invalid_arguments;
            dnnl_dim_t dense = 1;
            for (int d = got.ndims - 1; d >= 0; dense *= got.dims[d--])
                if (got.dims[d] > 1 && got.strides[d] != dense) return dnnl_invalid_arguments;
        }
        op = &settled;
    }
    bound_t bound;
    for (const auto &kv : op->args) {
        const dnnl_memory_t m = find(kv.first);
        if (m->is_host_scalar) return dnnl_invalid_arguments;
        auto &b = bound.t[bound.n++]; // (no kind has more than eight tensors)
        b.arg = kv.first;
        b.values = (char *)m->handles[0];
        b.offsets = nullptr;
        if (!b.values && !kv.second.has_zero_dim()) return dnnl_invalid_arguments;
        if (b.values) b.values += kv.second.offset0 * (dnnl_dim_t)dt_bits(kv.second.data_type) / 8;
        if (kv.second.is_grouped()) {
            if (!m->md.is_grouped() || !m->handles[1]) return dnnl_invalid_arguments;
            b.offsets = (const int *)m->handles[1];
        }
    }
    if (pd.engine->device < 0) {
        set_last_error("a device-less engine cannot execute primitives");
        return dnnl_runtime_error;
    }
    void *scratch = primitive.scratch;
    if (pd.scratch_bytes && pd.attr.scratchpad_mode == dnnl_scratchpad_mode_user) {
        dnnl_memory_t sp = find(DNNL_ARG_SCRATCHPAD);
        if (!sp || !sp->handles[0]) return dnnl_invalid_arguments;
        scratch = sp->handles[0];
        if (pd.kind >= dnnl_cuda_interop_rms_norm && (uintptr_t)scratch % 16) return dnnl_invalid_arguments; // (wide accesses)
    }
    cudaSetDevice(pd.engine->device);
    cudaEvent_t ev0 = nullptr, ev1 = nullptr;
    const bool verbose = verbose_level() >= 1;
    if (verbose) {
        cudaEventCreate(&ev0); cudaEventCreate(&ev1);
        cudaEventRecord(ev0, stream->stream);
    }
    profiling_begin(stream);
    const int rc = launch(primitive, pd.kind, *op, bound, scratch, stream->stream);
    profiling_end(stream);
    if (verbose) {
        cudaEventRecord(ev1, stream->stream);
        cudaEventSynchronize(ev1);
        float ms = 0;
        cudaEventElapsedTime(&ms, ev0, ev1);
        cudaEventDestroy(ev0); cudaEventDestroy(ev1);
        verbose_line("exec", pd, ms);
    }
    if (rc == 5) set_last_error(std::string("kernel launch: ") + cudaGetErrorString(cudaGetLastError()));
    return (dnnl_status_t)rc;
} catch (const std::bad_alloc &) {
    return dnnl_out_of_memory;
}

} // namespace qmm

extern "C" {

dnnl_status_t dnnl_cuda_interop_moe_route_primitive_desc_create(dnnl_primitive_desc_t *primitive_desc, dnnl_engine_t engine,
        const_dnnl_memory_desc_t logits_desc, const_dnnl_memory_desc_t weights_desc, const_dnnl_memory_desc_t indices_desc,
        dnnl_cuda_interop_scoring_t scoring, int normalize, float scale, const_dnnl_primitive_attr_t attr) {
    token_op_t op;
    op.scoring = (int)scoring; op.normalize = normalize != 0; op.scale = scale;
    return create(primitive_desc, engine, dnnl_cuda_interop_moe_route, op,
            {{DNNL_ARG_SRC, logits_desc}, {DNNL_ARG_DST, weights_desc}, {DNNL_ARG_DST_1, indices_desc}}, {}, attr);
}

dnnl_status_t dnnl_cuda_interop_moe_route_v2_primitive_desc_create(dnnl_primitive_desc_t *primitive_desc, dnnl_engine_t engine,
        const_dnnl_memory_desc_t logits_desc, const_dnnl_memory_desc_t bias_desc, const_dnnl_memory_desc_t weights_desc,
        const_dnnl_memory_desc_t indices_desc, dnnl_cuda_interop_scoring_t scoring, int normalize, float scale, int groups,
        int groups_kept, int group_best, const_dnnl_primitive_attr_t attr) {
    token_op_t op;
    op.scoring = (int)scoring; op.normalize = normalize != 0; op.scale = scale;
    op.groups = groups; op.groups_kept = groups_kept; op.group_best = group_best;
    return create(primitive_desc, engine, dnnl_cuda_interop_moe_route, op,
            {{DNNL_ARG_SRC, logits_desc}, {DNNL_ARG_DST, weights_desc}, {DNNL_ARG_DST_1, indices_desc}}, {{DNNL_ARG_BIAS, bias_desc}}, attr);
}

dnnl_status_t dnnl_cuda_interop_moe_route_backward_primitive_desc_create(dnnl_primitive_desc_t *primitive_desc,
        dnnl_engine_t engine, const_dnnl_memory_desc_t logits_desc, const_dnnl_memory_desc_t indices_desc,
        const_dnnl_memory_desc_t diff_weights_desc, const_dnnl_memory_desc_t diff_logits_desc,
        dnnl_cuda_interop_scoring_t scoring, int normalize, float scale, const_dnnl_primitive_attr_t attr) {
    token_op_t op;
    op.scoring = (int)scoring; op.normalize = normalize != 0; op.scale = scale;
    return create(primitive_desc, engine, dnnl_cuda_interop_moe_route_backward, op,
            {{DNNL_ARG_SRC, logits_desc}, {DNNL_ARG_SRC_1, indices_desc}, {DNNL_ARG_DIFF_DST, diff_weights_desc},
                    {DNNL_ARG_DIFF_SRC, diff_logits_desc}}, {}, attr);
}

dnnl_status_t dnnl_cuda_interop_moe_dispatch_primitive_desc_create(dnnl_primitive_desc_t *primitive_desc,
        dnnl_engine_t engine, const_dnnl_memory_desc_t src_desc, const_dnnl_memory_desc_t indices_desc,
        const_dnnl_memory_desc_t dst_desc, const_dnnl_memory_desc_t positions_desc, const_dnnl_primitive_attr_t attr) {
    return create(primitive_desc, engine, dnnl_cuda_interop_moe_dispatch, token_op_t(),
            {{DNNL_ARG_SRC, src_desc}, {DNNL_ARG_SRC_1, indices_desc}, {DNNL_ARG_DST, dst_desc}, {DNNL_ARG_DST_1, positions_desc}}, {}, attr);
}

dnnl_status_t dnnl_cuda_interop_moe_combine_primitive_desc_create(dnnl_primitive_desc_t *primitive_desc,
        dnnl_engine_t engine, const_dnnl_memory_desc_t src_desc, const_dnnl_memory_desc_t positions_desc,
        const_dnnl_memory_desc_t weights_desc, const_dnnl_memory_desc_t residual_desc, const_dnnl_memory_desc_t dst_desc,
        float dropout_p, const_dnnl_primitive_attr_t attr) {
    token_op_t op;
    op.p = dropout_p;
    return create(primitive_desc, engine, dnnl_cuda_interop_moe_combine, op,
            {{DNNL_ARG_SRC, src_desc}, {DNNL_ARG_SRC_1, positions_desc}, {DNNL_ARG_DST, dst_desc}},
            {{DNNL_ARG_WEIGHTS, weights_desc}, {DNNL_ARG_SRC_2, residual_desc}}, attr);
}

dnnl_status_t dnnl_cuda_interop_moe_combine_backward_primitive_desc_create(dnnl_primitive_desc_t *primitive_desc,
        dnnl_engine_t engine, const_dnnl_memory_desc_t diff_dst_desc, const_dnnl_memory_desc_t src_desc,
        const_dnnl_memory_desc_t positions_desc, const_dnnl_memory_desc_t weights_desc,
        const_dnnl_memory_desc_t diff_src_desc, const_dnnl_memory_desc_t diff_weights_desc, float dropout_p,
        const_dnnl_primitive_attr_t attr) {
    token_op_t op;
    op.p = dropout_p;
    return create(primitive_desc, engine, dnnl_cuda_interop_moe_combine_backward, op,
            {{DNNL_ARG_DIFF_DST, diff_dst_desc}, {DNNL_ARG_SRC, src_desc}, {DNNL_ARG_SRC_1, positions_desc},
                    {DNNL_ARG_WEIGHTS, weights_desc}, {DNNL_ARG_DIFF_SRC, diff_src_desc}, {DNNL_ARG_DIFF_WEIGHTS, diff_weights_desc}}, {}, attr);
}

dnnl_status_t dnnl_cuda_interop_dropout_primitive_desc_create(dnnl_primitive_desc_t *primitive_desc, dnnl_engine_t engine,
        const_dnnl_memory_desc_t src_desc, const_dnnl_memory_desc_t residual_desc, const_dnnl_memory_desc_t dst_desc,
        float p, const_dnnl_primitive_attr_t attr) {
    token_op_t op;
    op.p = p;
    return create(primitive_desc, engine, dnnl_cuda_interop_dropout, op,
            {{DNNL_ARG_SRC, src_desc}, {DNNL_ARG_DST, dst_desc}}, {{DNNL_ARG_SRC_2, residual_desc}}, attr);
}

dnnl_status_t dnnl_cuda_interop_rms_norm_primitive_desc_create(dnnl_primitive_desc_t *primitive_desc, dnnl_engine_t engine,
        const_dnnl_memory_desc_t src_desc, const_dnnl_memory_desc_t residual_desc, const_dnnl_memory_desc_t weights_desc,
        const_dnnl_memory_desc_t dst_desc, const_dnnl_memory_desc_t sum_desc, float epsilon, const_dnnl_primitive_attr_t attr) {
    token_op_t op;
    op.epsilon = epsilon;
    return create(primitive_desc, engine, dnnl_cuda_interop_rms_norm, op, {{DNNL_ARG_SRC, src_desc}, {DNNL_ARG_DST, dst_desc}},
            {{DNNL_ARG_SRC_2, residual_desc}, {DNNL_ARG_WEIGHTS, weights_desc}, {DNNL_ARG_DST_1, sum_desc}}, attr);
}

dnnl_status_t dnnl_cuda_interop_rms_norm_backward_primitive_desc_create(dnnl_primitive_desc_t *primitive_desc, dnnl_engine_t engine,
        const_dnnl_memory_desc_t diff_dst_desc, const_dnnl_memory_desc_t src_desc, const_dnnl_memory_desc_t weights_desc,
        const_dnnl_memory_desc_t diff_sum_desc, const_dnnl_memory_desc_t diff_src_desc, const_dnnl_memory_desc_t diff_weights_desc,
        float epsilon, const_dnnl_primitive_attr_t attr) {
    token_op_t op;
    op.epsilon = epsilon;
    return create(primitive_desc, engine, dnnl_cuda_interop_rms_norm_backward, op,
            {{DNNL_ARG_DIFF_DST, diff_dst_desc}, {DNNL_ARG_SRC, src_desc}, {DNNL_ARG_DIFF_SRC, diff_src_desc}},
            {{DNNL_ARG_WEIGHTS, weights_desc}, {DNNL_ARG_SRC_2, diff_sum_desc}, {DNNL_ARG_DIFF_WEIGHTS, diff_weights_desc}}, attr);
}

dnnl_status_t dnnl_cuda_interop_low_rank_adapter_primitive_desc_create(dnnl_primitive_desc_t *primitive_desc, dnnl_engine_t engine,
        const_dnnl_memory_desc_t src_desc, const_dnnl_memory_desc_t indices_desc, const_dnnl_memory_desc_t down_desc,
        const_dnnl_memory_desc_t up_desc, const_dnnl_memory_desc_t base_desc, const_dnnl_memory_desc_t dst_desc,
        const_dnnl_primitive_attr_t attr) {
    return create(primitive_desc, engine, dnnl_cuda_interop_low_rank_adapter, token_op_t(),
            {{DNNL_ARG_SRC, src_desc}, {DNNL_ARG_SRC_1, indices_desc}, {DNNL_ARG_WEIGHTS, down_desc}, {DNNL_ARG_WEIGHTS_1, up_desc},
                    {DNNL_ARG_DST, dst_desc}}, {{DNNL_ARG_SRC_2, base_desc}}, attr);
}

} // extern "C"
