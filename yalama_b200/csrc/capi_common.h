// Helpers of the kernel-level C ABI entry points: refusals and results with the calling thread's
// ylm_last_error(), pointer checks, the device's size.
#pragma once
#include "../../include/yalama_b200.h"
#include "ylm_kernels.h"

#include <cuda_runtime.h>

namespace ylm {

inline int refuse(int status, const char *why)
{
    set_last_error(why);
    return status;
}

inline int done(cudaError_t e)
{
    if (e == cudaSuccess)
    {
        set_last_error("");
        return YLM_OK;
    }
    // the runtime keeps a failed call's error until it is asked for, and a later launch of this library would
    // take it for its own
    cudaGetLastError();
    set_last_error(cudaGetErrorString(e));
    return YLM_CUDA_ERROR;
}

inline int no_device()
{
    cudaGetLastError();
    return refuse(YLM_CUDA_ERROR, "device set-up failed");
}

inline bool aligned(const void *p, uintptr_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

inline bool overlap(const void *a, size_t na, const void *b, size_t nb)
{
    const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
    return x < y + nb && y < x + na;
}

// SMs of the current device, 0 where it cannot be asked
inline int device_sms()
{
    int dev = 0, n = 0;
    if (cudaGetDevice(&dev) != cudaSuccess ||
        cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
        return 0;
    return n;
}

} // namespace ylm
