// ops_common.h -- what the host sides of the sequence operators share: argument checks, the device of a call, launches
#pragma once
#include <hip/hip_runtime.h>

#include <cstdint>
#include <cstring>

#include "../../include/helen_hip.h"
#include "error.h"

namespace helen {

// makes `device` current for a call and puts the caller's back
class OnDevice {
public:
    explicit OnDevice(int device) {
        if (hipGetDevice(&before_) != hipSuccess) before_ = device;
        status_ = before_ == device ? hipSuccess : hipSetDevice(device);
        moved_ = status_ == hipSuccess && before_ != device;
    }
    ~OnDevice() {
        if (moved_) (void)hipSetDevice(before_);
    }
    hipError_t status() const { return status_; }

private:
    int before_ = 0;
    bool moved_ = false;
    hipError_t status_ = hipSuccess;
};

inline int launched(const char* what) {
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? HELEN_OK : fail(HELEN_EHIP, "%s: launch failed: %s", what, hipGetErrorString(e));
}

inline int type_size(int dtype) { return dtype == HELEN_TYPE_FP32 ? 4 : 2; }
inline bool type_known(int dtype) { return dtype == HELEN_TYPE_FP32 || dtype == HELEN_TYPE_BF16 || dtype == HELEN_TYPE_FP16; }

// base and strides a multiple of `bytes`
inline bool aligned(const void* p, const int64_t* stride, int size, int bytes) {
    return (uintptr_t)p % bytes == 0 && stride[0] * size % bytes == 0 && stride[1] * size % bytes == 0;
}

// a 1-D grid of a x b workgroups of `threads`, and `more`: the runtime counts threads in 32 bits
inline bool grid_fits(int64_t a, int64_t b, int threads, int more = 0) {
    const int64_t most = ((int64_t(1) << 32) - 1) / threads - more;
    return a >= 0 && b >= 0 && (b == 0 || a <= most / b);
}

}  // namespace helen
