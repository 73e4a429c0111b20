// ops_delta.hip -- C entries of the gated delta rule (include/helen_hip.h): checks, workspace layout, forward launches
#include "ops_delta.h"

#include <initializer_list>

namespace helen {

namespace {

struct Carver {
    char* base;
    size_t at = 0;
    template <typename T>
    T* take(size_t count) {
        T* p = base ? (T*)(base + at) : nullptr;
        at += (count * sizeof(T) + 255) / 256 * 256;
        return p;
    }
};

// the forward call's workspace; with `keep` it goes on with what only the backward pass reads
size_t carve(const HelenDeltaRule& op, int keep, void* base, DeltaArgs* a) {
    Carver c{(char*)base};
    const size_t ks = (size_t)a->slots * a->hk, vs = (size_t)a->slots * a->hv;
    const int ni = op.dtype == HELEN_TYPE_BF16 ? 1 : (op.dtype == HELEN_TYPE_FP16 ? 2 : 3);
    const size_t rows = ks * (op.width_k / 8) * ni * 64, tri = vs * kTriFrags * 64;
    a->sink = c.take<float>(256);
    a->zeros = c.take<bf16x8>(3 * 64);
    const bool from_inputs = ni == 1 && !keep && !chains_are_few(*a);       // (delta_forward_kernel's InputRows)
    a->kf = from_inputs ? nullptr : c.take<bf16x8>(rows);
    a->ktf = c.take<bf16x8>(rows);
    a->qf = from_inputs ? nullptr : c.take<bf16x8>(rows);
    a->tf = c.take<bf16x8>(tri * 3);
    a->pf = c.take<bf16x8>(tri * 3);
    a->sc = c.take<float>(vs * 256);
    if (keep) {
        a->qtf = c.take<bf16x8>(rows);
        a->dots = c.take<f32x4>(ks * 10 * 128);
        a->ttf = c.take<bf16x8>(tri * 3);
        a->ptf = c.take<bf16x8>(tri * 3);
        a->states = c.take<float>(vs * op.width_k * op.width_v);
        a->e = c.take<float>(vs * kDeltaChunk * op.width_v);
    }
    return c.at;
}
size_t carve_backward(const HelenDeltaRule& op, void* base, DeltaArgs* a) {
    Carver c{(char*)base};
    const size_t vs = (size_t)a->slots * a->hv;
    a->dstates = c.take<float>(vs * op.width_k * op.width_v);
    a->z = c.take<float>(vs * kDeltaChunk * op.width_v);
    return c.at;
}

enum Check { kGeometry, kForward, kBackward };
int describe(const HelenDeltaRule* op, Check level, DeltaArgs* a) {
    const bool backward = level == kBackward;
    if (!op) return fail(HELEN_EINVAL, "delta rule: null description");
    if (op->struct_size != sizeof(HelenDeltaRule))
        return fail(HELEN_EINVAL, "delta rule: struct_size %zu, this library's is %zu", op->struct_size, sizeof(HelenDeltaRule));
    if (!type_known(op->dtype)) return fail(HELEN_EINVAL, "delta rule: unknown dtype %d", op->dtype);
    if (op->width_k != 64 && op->width_k != 128)
        return fail(HELEN_EINVAL, "delta rule: width_k %d is neither 64 nor 128", op->width_k);
    if (op->width_v < 64 || op->width_v > 256 || op->width_v % 64)
        return fail(HELEN_EINVAL, "delta rule: width_v %d is not 64, 128, 192 or 256", op->width_v);
    if (op->heads_k < 1 || op->heads_v < 1 || op->heads_v % op->heads_k)
        return fail(HELEN_EINVAL, "delta rule: %d value heads do not share %d key heads evenly", op->heads_v, op->heads_k);
    if (op->tokens < 0 || op->sequences < 1)
        return fail(HELEN_EINVAL, "delta rule: %d tokens in %d sequences", op->tokens, op->sequences);
    if (!op->offsets && op->tokens % op->sequences)
        return fail(HELEN_EINVAL, "delta rule: %d tokens are no %d sequences of one length", op->tokens, op->sequences);
    const int64_t slots = (int64_t)op->tokens / kDeltaChunk + op->sequences + 1;
    // launches: preparation and gradients by (slot, key head), chains by column groups of a state (256 threads where they are many)
    if (slots > INT32_MAX || !grid_fits(slots, op->heads_k, backward ? 4 * op->width_k : 256) ||
        !grid_fits(op->sequences, (int64_t)op->heads_v * (op->width_v / (16 * kColumnTiles)), 256, 7))
        return fail(HELEN_EINVAL, "delta rule: %d tokens x %d heads in %d sequences are more than one call takes", op->tokens,
                    op->heads_v, op->sequences);
    const int size = type_size(op->dtype);
    if (op->tokens > 0 && level != kGeometry) {
        if (!op->q || !op->k || !op->v || !op->g || !op->beta) return fail(HELEN_EINVAL, "delta rule: null input");
        if (!aligned(op->q, op->q_stride, size, 16) || !aligned(op->k, op->k_stride, size, 16) ||
            !aligned(op->v, op->v_stride, size, 16))
            return fail(HELEN_EINVAL, "delta rule: q, k, v and their strides must be multiples of 16 bytes");
        const int64_t most = int64_t(1) << 24;      // 64 rows fit 32 bits of elements
        for (const int64_t t : {op->q_stride[0], op->k_stride[0], op->v_stride[0], op->o ? op->o_stride[0] : 0, backward ? op->d_o_stride[0] : 0,
                                (int64_t)op->heads_v * op->width_v})
            if (t < 0 || t > most) return fail(HELEN_EINVAL, "delta rule: a stride of %lld elements between tokens", (long long)t);
        if (backward) {
            if (!op->d_o || !op->grad_q || !op->grad_k || !op->grad_v || !op->grad_g || !op->grad_beta)
                return fail(HELEN_EINVAL, "delta rule: null gradient");
            if (!aligned(op->d_o, op->d_o_stride, size, 16))
                return fail(HELEN_EINVAL, "delta rule: d_o and its strides must be multiples of 16 bytes");
        }
    }
    memset(a, 0, sizeof(*a));
    a->q = op->q; a->k = op->k; a->v = op->v; a->g = op->g; a->beta = op->beta; a->offsets = op->offsets;
    a->s0 = op->initial_state; a->s1 = op->final_state; a->o = op->o;
    a->q_t = op->q_stride[0]; a->q_h = op->q_stride[1]; a->k_t = op->k_stride[0]; a->k_h = op->k_stride[1];
    a->v_t = op->v_stride[0]; a->v_h = op->v_stride[1]; a->o_t = op->o_stride[0]; a->o_h = op->o_stride[1];
    a->g_t = op->g_stride[0]; a->g_h = op->g_stride[1]; a->b_t = op->beta_stride[0]; a->b_h = op->beta_stride[1];
    a->tokens = op->tokens; a->nseq = op->sequences; a->seq_len = op->tokens / op->sequences;
    a->hk = op->heads_k; a->hv = op->heads_v; a->group = op->heads_v / op->heads_k; a->dv_width = op->width_v;
    a->slots = (int)slots; a->scale = op->scale; a->zero_tail = op->zero_tail != 0;
    if (backward) {
        a->dout = op->d_o; a->do_t = op->d_o_stride[0]; a->do_h = op->d_o_stride[1];
        a->ds1 = op->d_final_state; a->ds0 = op->grad_initial_state;
        a->dq = op->grad_q; a->dk = op->grad_k; a->dv = op->grad_v; a->dg = op->grad_g; a->dbeta = op->grad_beta;
    }
    return HELEN_OK;
}

template <typename In, int DK, bool KEEP>
void launch_forward(const DeltaArgs& a, hipStream_t s) {
    if (a.tokens > 0) hipLaunchKernelGGL((delta_prep_kernel<In, DK, KEEP>), dim3((unsigned)a.slots * a.hk), dim3(256), 0, s, a);
    if (chains_are_few(a)) hipLaunchKernelGGL((delta_forward_long_kernel<In, DK, KEEP>), dim3(chain_grid(a, 16)), dim3(512), 0, s, a);
    else hipLaunchKernelGGL((delta_forward_kernel<In, DK, KEEP>), dim3(chain_grid(a, 16 * kColumnTiles)), dim3(256), 0, s, a);
}
template <typename In, int DK>
void launch_forward(const DeltaArgs& a, int keep, hipStream_t s) {
    keep ? launch_forward<In, DK, true>(a, s) : launch_forward<In, DK, false>(a, s);
}

}  // namespace

}  // namespace helen

using namespace helen;

extern "C" {

int helen_delta_rule_bytes(const HelenDeltaRule* op, size_t* forward_bytes, size_t* kept_bytes, size_t* backward_bytes) {
    DeltaArgs a;
    if (const int rc = describe(op, kGeometry, &a)) return rc;
    if (forward_bytes) *forward_bytes = carve(*op, 0, nullptr, &a);
    if (kept_bytes) *kept_bytes = carve(*op, 1, nullptr, &a);
    if (backward_bytes) *backward_bytes = carve_backward(*op, nullptr, &a);
    return HELEN_OK;
}

int helen_delta_rule_forward(const HelenDeltaRule* op, int keep, void* workspace, size_t workspace_bytes, void* stream) {
    DeltaArgs a;
    if (const int rc = describe(op, kForward, &a)) return rc;
    const size_t need = carve(*op, keep != 0, workspace, &a);
    if (workspace_bytes < need || !workspace || (uintptr_t)workspace % 256)
        return fail(HELEN_EINVAL, "delta rule: workspace of %zu bytes, %zu are needed, 256-byte aligned", workspace_bytes, need);
    if (!a.o) {          // the chain stores its rows all the same: into the sink
        a.o = a.sink;
        a.o_t = a.o_h = a.zero_tail = 0;
    }
    OnDevice on(op->device);
    if (on.status() != hipSuccess) return fail(HELEN_ENODEV, "delta rule: device %d: %s", op->device, hipGetErrorString(on.status()));
    hipStream_t s = (hipStream_t)stream;
    switch (op->dtype) {
        case HELEN_TYPE_BF16:
            if (op->width_k == 64) launch_forward<InBf16, 64>(a, keep, s); else launch_forward<InBf16, 128>(a, keep, s);
            break;
        case HELEN_TYPE_FP16:
            if (op->width_k == 64) launch_forward<InF16, 64>(a, keep, s); else launch_forward<InF16, 128>(a, keep, s);
            break;
        default:
            if (op->width_k == 64) launch_forward<InF32, 64>(a, keep, s); else launch_forward<InF32, 128>(a, keep, s);
    }
    return launched("delta rule forward");
}

int helen_delta_rule_backward(const HelenDeltaRule* op, const void* kept, size_t kept_bytes, void* workspace,
                              size_t workspace_bytes, void* stream) {
    DeltaArgs a;
    if (const int rc = describe(op, kBackward, &a)) return rc;
    const size_t keep_need = carve(*op, 1, (void*)kept, &a), need = carve_backward(*op, workspace, &a);
    if (!kept || kept_bytes < keep_need || (uintptr_t)kept % 256)
        return fail(HELEN_EINVAL, "delta rule: kept workspace of %zu bytes, the forward call's has %zu, 256-byte aligned", kept_bytes,
                    keep_need);
    if (!workspace || workspace_bytes < need || (uintptr_t)workspace % 256)
        return fail(HELEN_EINVAL, "delta rule: workspace of %zu bytes, %zu are needed, 256-byte aligned", workspace_bytes, need);
    OnDevice on(op->device);
    if (on.status() != hipSuccess) return fail(HELEN_ENODEV, "delta rule: device %d: %s", op->device, hipGetErrorString(on.status()));
    delta_backward_launch(op->dtype, op->width_k, a, (hipStream_t)stream);
    return launched("delta rule backward");
}

}  // extern "C"
