// What the C-ABI front ends share: the calling thread's error text and the device guard.
#pragma once

#include <cuda_runtime.h>

namespace exb {

// Stores the text of the calling thread's last error and returns `code` (defined in exb_api.cu).
int fail(int code, const char *fmt, ...);

// Makes `device` current for the duration of one entry point and restores the
// previous device afterwards (the reference calls cudaSetDevice without
// restoring, cuda/bindings.cu:45).
struct DeviceGuard {
    int prev = -1;
    bool ok = true;
    explicit DeviceGuard(int device)
    {
        if (cudaGetDevice(&prev) != cudaSuccess) { ok = false; return; }
        if (device >= 0 && device != prev && cudaSetDevice(device) != cudaSuccess) ok = false;
    }
    ~DeviceGuard()
    {
        int cur = -1;
        if (prev >= 0 && cudaGetDevice(&cur) == cudaSuccess && cur != prev) cudaSetDevice(prev);
    }
};

}  // namespace exb
