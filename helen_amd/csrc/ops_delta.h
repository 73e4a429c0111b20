// ops_delta.h -- the delta rule's launches, over the sources they are compiled in
#pragma once
#include "kernels_delta.h"
#include "ops_common.h"

namespace helen {

void delta_backward_launch(int dtype, int width_k, const DeltaArgs& a, hipStream_t s);

}  // namespace helen
