// Host-side helpers shared by the translation units of the library: the error text and its macros.
#pragma once
#include <hip/hip_runtime.h>

#include "../../include/wino_amd.h"

namespace wino {

// records the text that wino_last_error() returns on this thread; returns `code`
__attribute__((visibility("hidden"))) int fail(int code, const char* fmt, ...);

// compute units of the current device
__attribute__((visibility("hidden"))) int device_cus();

#define HIP_TRY(expr)                                                                                   \
    do {                                                                                                \
        hipError_t e_ = (expr);                                                                         \
        if (e_ != hipSuccess) return wino::fail(WINO_ERR_HIP, "%s: %s", #expr, hipGetErrorString(e_)); \
    } while (0)

#define LAUNCH_CHECK(name)                                                                                     \
    do {                                                                                                       \
        hipError_t e_ = hipGetLastError();                                                                     \
        if (e_ != hipSuccess) return wino::fail(WINO_ERR_HIP, "launch %s: %s", name, hipGetErrorString(e_)); \
    } while (0)

}  // namespace wino
