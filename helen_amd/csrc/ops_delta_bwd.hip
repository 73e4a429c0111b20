// ops_delta_bwd.hip -- launches of the gated delta rule's backward pass
#include "kernels_delta_bwd.h"
#include "ops_delta.h"

namespace helen {

namespace {

template <typename In, int DK>
void launch(const DeltaArgs& a, hipStream_t s) {
    if (chains_are_few(a)) hipLaunchKernelGGL((delta_backward_long_kernel<In, DK>), dim3(chain_grid(a, 16)), dim3(512), 0, s, a);
    else hipLaunchKernelGGL((delta_backward_kernel<In, DK>), dim3(chain_grid(a, 16 * kColumnTiles)), dim3(256), 0, s, a);
    if (a.tokens == 0) return;
    const dim3 chunks((unsigned)a.slots * a.hk), block(DK * 4);
    if (a.group == 1) hipLaunchKernelGGL((delta_grads_kernel<In, DK, false>), chunks, block, 0, s, a);
    else hipLaunchKernelGGL((delta_grads_kernel<In, DK, true>), chunks, block, 0, s, a);
}

}  // namespace

void delta_backward_launch(int dtype, int width_k, const DeltaArgs& a, hipStream_t s) {
    switch (dtype) {
        case HELEN_TYPE_BF16: width_k == 64 ? launch<InBf16, 64>(a, s) : launch<InBf16, 128>(a, s); break;
        case HELEN_TYPE_FP16: width_k == 64 ? launch<InF16, 64>(a, s) : launch<InF16, 128>(a, s); break;
        default: width_k == 64 ? launch<InF32, 64>(a, s) : launch<InF32, 128>(a, s);
    }
}

}  // namespace helen
