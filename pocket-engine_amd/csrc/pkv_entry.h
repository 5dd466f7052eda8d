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

// Strides of rows of 16-byte pieces: multiples of 8 elements, 0 .. 2^24.
inline bool stride_ok(int64_t s) { return s >= 0 && s % 8 == 0 && s <= ((int64_t)1 << 24); }

// T rows of H heads of D elements that are written lie apart: the heads inside
// a row's stride or the rows inside a head's.
inline bool apart(int64_t row, int64_t head, int T, int H, int D) {
    const bool rows = T <= 1 || row >= D, heads = H <= 1 || head >= D;
    return rows && heads && (T <= 1 || H <= 1 || row >= (H - 1) * head + D || head >= (T - 1) * row + D);
}

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
