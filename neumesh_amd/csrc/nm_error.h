// nm_error.h -- error reporting shared by the library's translation units (nm_api.hip, nm_dense.hip, nm_scan.hip).
#pragma once

#include <hip/hip_runtime.h>

// stores a thread-local message for nm_last_error() and returns 1 (defined in nm_api.hip)
__attribute__((visibility("hidden"))) int nm_fail(const char* fmt, ...);

#define NM_HIP(call)                                                                          \
    do {                                                                                      \
        hipError_t e_ = (call);                                                               \
        if (e_ != hipSuccess) return nm_fail("%s failed: %s", #call, hipGetErrorString(e_));  \
    } while (0)
#define NM_LAUNCH_CHECK()                                                                      \
    do {                                                                                       \
        hipError_t e_ = hipGetLastError();                                                     \
        if (e_ != hipSuccess) return nm_fail("kernel launch failed: %s", hipGetErrorString(e_)); \
    } while (0)
