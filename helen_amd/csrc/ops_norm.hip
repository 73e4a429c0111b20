// ops_norm.hip -- C entries of the delta rule's single-token form and of layer norm (include/helen_hip.h)
#include "kernels_delta_step.h"
#include "kernels_norm.h"
#include "ops_common.h"

using namespace helen;

namespace {

template <typename In>
void launch_step(const DeltaStepArgs& a, int width_k, hipStream_t s) {
    const dim3 grid((unsigned)a.rows * a.hv * (a.dv_width / 64));
    if (width_k == 64) hipLaunchKernelGGL((delta_step_kernel<In, 64>), grid, dim3(256), 0, s, a);
    else hipLaunchKernelGGL((delta_step_kernel<In, 128>), grid, dim3(256), 0, s, a);
}

// Lanes per row and 16-byte pieces a lane holds: the narrowest pair that takes a row; 0: the wide kernels.  Forward / backward in us
// against wider pairs: 262143 x 128 bf16 (16, 1) 23 / 44, (16, 2) 29 / 54, (64, 1) 66 / 88; 100000 x 512 fp16 (64, 1) 36 / 57, (64, 2)
// 43 / 98, (256, 1) 98 / 117; 32000 x 2048 bf16 (256, 1) 44 / 86, (256, 2) 58 / 129.
struct NormPlan {
    int lanes, pieces;
};
NormPlan norm_plan(int width, int dtype) {
    const int per = 16 / type_size(dtype), pieces = (width + per - 1) / per;
    if (pieces <= 16) return {16, 1};
    if (pieces <= 32) return {16, 2};
    if (pieces <= 64) return {64, 1};
    if (pieces <= 128) return {64, 2};
    if (pieces <= 256) return {256, 1};
    if (pieces <= 512) return {256, 2};
    if (pieces <= 1024) return {256, 4};
    return {0, 0};
}
// strips of columns of the wide kernels' second backward pass
int norm_strips(int width, int dtype) {
    const int per = 256 * (16 / type_size(dtype));
    return (width + per - 1) / per;
}
// Workgroups of a pass.  Forward: more rows in flight against one load of the weight; 32000 x 2048 bf16 44 us with 2048, 42.4 with
// 4096, 41.2 with 8192, but 8192 x 8192 44 with 4096 and 47.5 with 8192, where none has a second row.  Backward: each writes
// one partial sum of the weight's gradient and the second kernel reads it; 32000 x 2048 bf16 109 us with 256, 78 with 512, 87 with
// 1024, 96 with 2048, and 262143 x 128 43, 37, 45, 42.  The wide kernels: 2048 with their strips.
constexpr int kNormForwardGroups = 4096, kNormBackwardGroups = 512, kNormWideGroups = 2048;
int norm_groups(const HelenLayerNorm& op, bool backward) {
    const NormPlan p = norm_plan(op.width, op.dtype);
    const int64_t rows = p.lanes ? 256 / p.lanes : 1, all = (op.rows + rows - 1) / rows;
    const int strips = norm_strips(op.width, op.dtype);
    const int most = !backward ? kNormForwardGroups : (p.lanes ? kNormBackwardGroups : (kNormWideGroups + strips - 1) / strips);
    return (int)(all < most ? (all > 0 ? all : 1) : most);
}
size_t norm_backward_bytes(const HelenLayerNorm& op) {
    const bool wide = !norm_plan(op.width, op.dtype).lanes;
    return ((size_t)norm_groups(op, true) * 2 * op.width + (wide ? 2 * (size_t)op.rows : 0)) * sizeof(float);
}

int check(const HelenLayerNorm* op, bool backward) {
    if (!op) return fail(HELEN_EINVAL, "layer norm: null description");
    if (op->struct_size != sizeof(HelenLayerNorm))
        return fail(HELEN_EINVAL, "layer norm: struct_size %zu, this library's is %zu", op->struct_size, sizeof(HelenLayerNorm));
    if (!type_known(op->dtype) || !type_known(op->weight_dtype))
        return fail(HELEN_EINVAL, "layer norm: unknown dtype %d / %d", op->dtype, op->weight_dtype);
    if (op->weight_dtype != op->dtype && op->weight_dtype != HELEN_TYPE_FP32)
        return fail(HELEN_EINVAL, "layer norm: the weight is of the input's type or float32");
    if (op->width < 1 || op->rows < 0 || op->width > (1 << 28))
        return fail(HELEN_EINVAL, "layer norm: %lld rows of width %d", (long long)op->rows, op->width);
    if (!(op->eps >= 0.f)) return fail(HELEN_EINVAL, "layer norm: eps %g", (double)op->eps);
    // a workgroup a row only in the wide kernels; the others' bound is what mean and rstd could be stored for
    const bool wide = !norm_plan(op->width, op->dtype).lanes;
    if (wide ? !grid_fits(op->rows, 1, 256) : op->rows >= int64_t(1) << 36)
        return fail(HELEN_EINVAL, "layer norm: %lld rows of width %d are more than one call takes", (long long)op->rows, op->width);
    if (op->rows > 0) {
        if (!op->x || (!backward && !op->y)) return fail(HELEN_EINVAL, "layer norm: null input or output");
        if (backward && (!op->dy || !op->dx || !op->mean || !op->rstd)) return fail(HELEN_EINVAL, "layer norm: null input or output");
    }
    return HELEN_OK;
}
NormArgs args_of(const HelenLayerNorm& op) {
    NormArgs a;
    memset(&a, 0, sizeof(a));
    a.x = op.x; a.w = op.weight; a.b = op.bias; a.dy = op.dy; a.y = op.y; a.dx = op.dx; a.dw = op.dweight; a.db = op.dbias;
    a.mean = op.mean; a.rstd = op.rstd; a.rows = op.rows; a.x_t = op.x_stride; a.y_t = op.y_stride; a.dy_t = op.dy_stride;
    a.dx_t = op.dx_stride; a.width = op.width; a.eps = op.eps;
    return a;
}

template <typename In, typename W>
void launch_norm(const NormArgs& a, int dtype, bool backward, hipStream_t s) {
    const NormPlan p = norm_plan(a.width, dtype);
    const dim3 block(256);
    const dim3 grid((unsigned)a.groups);
#define HELEN_NORM(L, NV)                                                                                            \
    if (p.lanes == L && p.pieces == NV) {                                                                            \
        if (backward) hipLaunchKernelGGL((norm_backward_kernel<In, W, L, NV>), grid, block, 0, s, a);             \
        else hipLaunchKernelGGL((norm_forward_kernel<In, W, L, NV>), grid, block, 0, s, a);                       \
        return;                                                                                                      \
    }
    HELEN_NORM(16, 1)
    HELEN_NORM(16, 2)
    HELEN_NORM(64, 1)
    HELEN_NORM(64, 2)
    HELEN_NORM(256, 1)
    HELEN_NORM(256, 2)
    HELEN_NORM(256, 4)
#undef HELEN_NORM
    if (!backward) {
        hipLaunchKernelGGL((norm_forward_wide_kernel<In, W>), dim3((unsigned)a.rows), block, 0, s, a);
        return;
    }
    if (a.rows > 0) hipLaunchKernelGGL((norm_backward_sums_kernel<In, W>), dim3((unsigned)a.rows), block, 0, s, a);
    hipLaunchKernelGGL((norm_backward_strip_kernel<In, W>), dim3((unsigned)norm_strips(a.width, dtype), (unsigned)a.groups), block, 0, s, a);
}
void launch_norm(const HelenLayerNorm& op, const NormArgs& a, bool backward, hipStream_t s) {
    const bool f32w = op.weight_dtype == HELEN_TYPE_FP32;
    switch (op.dtype) {
        case HELEN_TYPE_BF16: f32w ? launch_norm<InBf16, InF32>(a, op.dtype, backward, s) : launch_norm<InBf16, InBf16>(a, op.dtype, backward, s); break;
        case HELEN_TYPE_FP16: f32w ? launch_norm<InF16, InF32>(a, op.dtype, backward, s) : launch_norm<InF16, InF16>(a, op.dtype, backward, s); break;
        default: launch_norm<InF32, InF32>(a, op.dtype, backward, s);
    }
}
template <typename W>
void launch_reduce(const NormArgs& a, hipStream_t s) {
    const unsigned strips = (2u * a.width + 31) / 32, most = 1u << 20;       // (threads of a launch are counted in 32 bits)
    hipLaunchKernelGGL(norm_reduce_kernel<W>, dim3(strips < most ? strips : most), dim3(1024), 0, s, a);
}

}  // namespace

extern "C" {

int helen_delta_rule_step(const HelenDeltaStep* op, void* stream) {
    if (!op) return fail(HELEN_EINVAL, "delta step: null description");
    if (op->struct_size != sizeof(HelenDeltaStep))
        return fail(HELEN_EINVAL, "delta step: struct_size %zu, this library's is %zu", op->struct_size, sizeof(HelenDeltaStep));
    if (!type_known(op->dtype)) return fail(HELEN_EINVAL, "delta step: unknown dtype %d", op->dtype);
    if (op->width_k != 64 && op->width_k != 128)
        return fail(HELEN_EINVAL, "delta step: width_k %d is neither 64 nor 128", op->width_k);
    if (op->width_v < 64 || op->width_v > 256 || op->width_v % 64)
        return fail(HELEN_EINVAL, "delta step: width_v %d is not 64, 128, 192 or 256", op->width_v);
    if (op->heads_k < 1 || op->heads_v < 1 || op->heads_v % op->heads_k)
        return fail(HELEN_EINVAL, "delta step: %d value heads do not share %d key heads evenly", op->heads_v, op->heads_k);
    if (op->rows < 0 || op->pool < 0 || (!op->slots && op->rows > op->pool))
        return fail(HELEN_EINVAL, "delta step: %d rows over a pool of %d states", op->rows, op->pool);
    if (op->rows == 0) return HELEN_OK;
    if (!grid_fits(op->rows, (int64_t)op->heads_v * (op->width_v / 64), 256))
        return fail(HELEN_EINVAL, "delta step: %d rows x %d heads are more than one call takes", op->rows, op->heads_v);
    if (!op->q || !op->k || !op->v || !op->g || !op->beta || !op->o || (!op->state && op->pool > 0))
        return fail(HELEN_EINVAL, "delta step: null input or output");
    const int size = type_size(op->dtype);
    if (!aligned(op->v, op->v_stride, size, 4 * size)) return fail(HELEN_EINVAL, "delta step: v and its strides must be multiples of four elements");
    if ((uintptr_t)op->state % 16 || op->state_stride % 4 ||
        op->state_stride < (int64_t)op->heads_v * op->width_k * op->width_v)
        return fail(HELEN_EINVAL, "delta step: state not 16-byte aligned, or its stride %lld overlaps", (long long)op->state_stride);
    OnDevice on(op->device);
    if (on.status() != hipSuccess) return fail(HELEN_ENODEV, "delta step: device %d: %s", op->device, hipGetErrorString(on.status()));
    DeltaStepArgs a;
    memset(&a, 0, sizeof(a));
    a.q = op->q; a.k = op->k; a.v = op->v; a.g = op->g; a.beta = op->beta; a.slots = op->slots; a.state = op->state; a.o = op->o;
    a.q_t = op->q_stride[0]; a.q_h = op->q_stride[1]; a.k_t = op->k_stride[0]; a.k_h = op->k_stride[1];
    a.v_t = op->v_stride[0]; a.v_h = op->v_stride[1]; a.o_t = op->o_stride[0]; a.o_h = op->o_stride[1];
    a.g_t = op->g_stride[0]; a.g_h = op->g_stride[1]; a.b_t = op->beta_stride[0]; a.b_h = op->beta_stride[1];
    a.s_t = op->state_stride; a.rows = op->rows; a.pool = op->pool; a.hk = op->heads_k; a.hv = op->heads_v;
    a.group = op->heads_v / op->heads_k; a.dv_width = op->width_v; a.scale = op->scale;
    hipStream_t s = (hipStream_t)stream;
    switch (op->dtype) {
        case HELEN_TYPE_BF16: launch_step<InBf16>(a, op->width_k, s); break;
        case HELEN_TYPE_FP16: launch_step<InF16>(a, op->width_k, s); break;
        default: launch_step<InF32>(a, op->width_k, s);
    }
    return launched("delta step");
}

int helen_layer_norm_forward(const HelenLayerNorm* op, void* stream) {
    if (const int rc = check(op, false)) return rc;
    if (op->rows == 0) return HELEN_OK;
    OnDevice on(op->device);
    if (on.status() != hipSuccess) return fail(HELEN_ENODEV, "layer norm: device %d: %s", op->device, hipGetErrorString(on.status()));
    NormArgs a = args_of(*op);
    a.groups = norm_groups(*op, false);
    launch_norm(*op, a, false, (hipStream_t)stream);
    return launched("layer norm forward");
}

int helen_layer_norm_bytes(const HelenLayerNorm* op, size_t* backward_bytes) {
    if (!op || op->struct_size != sizeof(HelenLayerNorm)) return fail(HELEN_EINVAL, "layer norm: null or foreign description");
    if (!backward_bytes) return fail(HELEN_EINVAL, "layer norm: null output");
    if (!type_known(op->dtype) || op->width < 1 || op->rows < 0) return fail(HELEN_EINVAL, "layer norm: %lld rows of width %d", (long long)op->rows, op->width);
    *backward_bytes = norm_backward_bytes(*op);
    return HELEN_OK;
}

int helen_layer_norm_backward(const HelenLayerNorm* op, void* workspace, size_t workspace_bytes, void* stream) {
    if (const int rc = check(op, true)) return rc;
    NormArgs a = args_of(*op);
    a.groups = norm_groups(*op, true);
    const size_t need = norm_backward_bytes(*op);
    if (!workspace || workspace_bytes < need || (uintptr_t)workspace % 16)
        return fail(HELEN_EINVAL, "layer norm: workspace of %zu bytes, %zu are needed, 16-byte aligned", workspace_bytes, need);
    a.partial = (float*)workspace;
    a.sums = a.partial + (size_t)a.groups * 2 * op->width;
    OnDevice on(op->device);
    if (on.status() != hipSuccess) return fail(HELEN_ENODEV, "layer norm: device %d: %s", op->device, hipGetErrorString(on.status()));
    hipStream_t s = (hipStream_t)stream;
    launch_norm(*op, a, true, s);
    if (op->dweight || op->dbias) {
        switch (op->weight_dtype) {
            case HELEN_TYPE_BF16: launch_reduce<InBf16>(a, s); break;
            case HELEN_TYPE_FP16: launch_reduce<InF16>(a, s); break;
            default: launch_reduce<InF32>(a, s);
        }
    }
    return launched("layer norm backward");
}

}  // extern "C"
