// What the translation units of the C ABI share: the context, the calling
// thread's last error, and small argument checks.
#pragma once
#include "../../include/dyninfer_mi355x.h"

#include <hip/hip_runtime.h>

#include <string>

// A context: the device it was opened on and that device's copy of `scratch`.
// Immutable after dyninfer_mi355x_open, so calls from any number of threads
// share it without locks; each call's temporary lives in the caller's
// workspace (or, for the no-allocation entry point, in `scratch`).
struct dyninfer_mi355x_ctx {
    int device;
    uint8_t* scratch;
};

namespace dmx {

inline thread_local std::string g_last_error;

inline int fail(int code, const std::string& msg) {
    g_last_error = msg;
    return code;
}

inline int hip_fail(hipError_t e, const char* what) {
    return fail(DYNINFER_MI355X_ERR_HIP, std::string(what) + ": " + hipGetErrorName(e) + ": " + hipGetErrorString(e));
}

inline bool aligned(const void* p, uintptr_t a) { return ((uintptr_t)p & (a - 1)) == 0; }

// Makes ctx->device current for the duration of a call, restoring the caller's.
struct DeviceGuard {
    int prev = -1;
    hipError_t err = hipSuccess;
    explicit DeviceGuard(int dev) {
        err = hipGetDevice(&prev);
        if (err == hipSuccess && prev != dev) err = hipSetDevice(dev);
    }
    ~DeviceGuard() {
        int cur = -1;
        if (prev >= 0 && hipGetDevice(&cur) == hipSuccess && cur != prev) (void)hipSetDevice(prev);
    }
};

inline int check_ctx(dyninfer_mi355x_ctx_t* ctx) {
    if (!ctx) return fail(DYNINFER_MI355X_ERR_INVALID_ARGUMENT, "context is NULL");
    return 0;
}

}  // namespace dmx
