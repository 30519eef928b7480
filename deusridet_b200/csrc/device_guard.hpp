// device_guard.hpp — makes a device current for one call and puts the caller's back.
#pragma once

#include <cuda_runtime.h>

namespace drkv {

class DeviceGuard {
public:
    explicit DeviceGuard(int device) {
        ok_ = cudaGetDevice(&prev_) == cudaSuccess;
        if (ok_ && prev_ != device) {
            ok_ = cudaSetDevice(device) == cudaSuccess;
            changed_ = ok_;
        }
        if (!ok_) cudaGetLastError();   // reported by ok(): not left behind for the caller's next CUDA call
    }
    ~DeviceGuard() {
        if (changed_) cudaSetDevice(prev_);
    }
    DeviceGuard(const DeviceGuard&) = delete;
    DeviceGuard& operator=(const DeviceGuard&) = delete;
    bool ok() const { return ok_; }

private:
    int prev_ = 0;
    bool ok_ = false, changed_ = false;
};

}  // namespace drkv
