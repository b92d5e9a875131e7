// The opt-in to more than 48 KB of dynamic shared memory, a kernel's on each
// device: asked for once.
#pragma once
#include <cuda_runtime.h>

#include "common.cuh"

namespace nsb {

// `most`: the caller's, one a kernel, zero at first. What is asked for is always
// all that a block may have, so that two threads at once set the same.
template <typename F>
bool allow_shared(F kernel, size_t bytes, size_t (&most)[kMaxDevices]) {
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) return false;
    if (bytes <= most[dev]) return true;
    int limit = 0;
    if (cudaDeviceGetAttribute(&limit, cudaDevAttrMaxSharedMemoryPerBlockOptin, dev) != cudaSuccess) return false;
    cudaFuncAttributes at;
    if (cudaFuncGetAttributes(&at, kernel) != cudaSuccess) return false;
    limit -= (int)at.sharedSizeBytes;
    if ((long long)bytes > limit ||
        cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, limit) != cudaSuccess)
        return false;
    most[dev] = limit;
    return true;
}

}  // namespace nsb
