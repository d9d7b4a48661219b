// What the C-ABI translation units share: the thread's error message, argument and pointer checks, and the
// device guard of the entry points.
#pragma once
#include <cuda_runtime.h>

#include <cstdarg>
#include <cstdint>
#include <cstdio>

#include "../../include/bms_b200.h"

namespace bms {

constexpr int kMaxDevices = 64;

inline thread_local char g_error[512] = "";

inline int fail(int code, const char* fmt, ...) {
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(g_error, sizeof g_error, fmt, ap);
    va_end(ap);
    return code;
}

inline int cuda_fail(cudaError_t e, const char* what) {
    cudaGetLastError();  // clear a non-sticky error so later calls start clean
    return fail(BMS_ERROR_CUDA, "%s: %s", what, cudaGetErrorString(e));
}

#define BMS_CUDA(call, what)                                  \
    do {                                                      \
        const cudaError_t e_ = (call);                        \
        if (e_ != cudaSuccess) return cuda_fail(e_, (what));  \
    } while (0)

struct DeviceGuard {
    int prev = -1, want = -1;
    cudaError_t enter(int device) {
        want = device;
        cudaError_t e = cudaGetDevice(&prev);
        if (e != cudaSuccess) return e;
        if (prev != device) return cudaSetDevice(device);
        return cudaSuccess;
    }
    ~DeviceGuard() {
        if (prev >= 0 && prev != want) cudaSetDevice(prev);
    }
};

inline int check_device(int device) {
    int n = 0;
    BMS_CUDA(cudaGetDeviceCount(&n), "cudaGetDeviceCount");
    if (device < 0 || device >= n) return fail(BMS_ERROR_INVALID_ARGUMENT, "invalid CUDA device %d", device);
    return BMS_SUCCESS;
}

// Every pointer the kernels touch must be device (or managed) memory of `device`.
inline int check_ptr(const void* p, int device, const char* name, size_t align) {
    if (p == nullptr) return fail(BMS_ERROR_INVALID_ARGUMENT, "%s must not be NULL", name);
    if (reinterpret_cast<uintptr_t>(p) % align != 0)
        return fail(BMS_ERROR_INVALID_ARGUMENT, "%s must be %zu-byte aligned", name, align);
    cudaPointerAttributes a;
    const cudaError_t e = cudaPointerGetAttributes(&a, p);
    if (e != cudaSuccess) {
        cudaGetLastError();
        return fail(BMS_ERROR_INVALID_ARGUMENT, "%s is not a CUDA pointer", name);
    }
    if (a.type != cudaMemoryTypeDevice && a.type != cudaMemoryTypeManaged)
        return fail(BMS_ERROR_INVALID_ARGUMENT, "%s must be CUDA device memory", name);
    if (a.device != device)
        return fail(BMS_ERROR_INVALID_ARGUMENT, "%s is on device %d, expected device %d", name, a.device, device);
    return BMS_SUCCESS;
}

#define BMS_CHECK(expr)                      \
    do {                                     \
        const int rc_ = (expr);              \
        if (rc_ != BMS_SUCCESS) return rc_;  \
    } while (0)

}  // namespace bms
