// What the files with C-ABI entry points share on the host.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/pkv.h"

namespace {

inline int status_of(hipError_t e) { return e == hipSuccess ? PKV_OK : (int)e; }

inline int launch_status() { return status_of(hipGetLastError()); }

inline bool aligned(const void* p, size_t a) { return ((uintptr_t)p % a) == 0; }

}  // namespace
