// What the files with C-ABI entry points share on the host.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <atomic>

#include "../../include/pkv.h"

namespace {

inline int status_of(hipError_t e) { return e == hipSuccess ? PKV_OK : (int)e; }

inline int launch_status() { return status_of(hipGetLastError()); }

inline bool aligned(const void* p, size_t a) { return ((uintptr_t)p % a) == 0; }

// Compute units of the current device, cached per device.
inline int device_cus() {
    static std::atomic<int> cus[64];
    int dev = 0;
    if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) return 256;
    int n = cus[dev].load(std::memory_order_relaxed);
    if (n == 0) {
        if (hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || n <= 0) n = 256;
        cus[dev].store(n, std::memory_order_relaxed);
    }
    return n;
}

}  // namespace
