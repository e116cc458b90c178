// device_check.hpp — argument checks shared by the C entry points.
#pragma once

#include "common.cuh"

namespace aaedn_dev
{

// Rejects pointers that are null, misaligned or not memory of the current
// device (its kernels could not, or would slowly, reach them).
inline int check_device_ptr(const char* fn, const void* p, const char* what, size_t align)
{
    if (!p)
        return set_error(AAEDN_EINVAL, "%s: %s is null", fn, what);
    if (reinterpret_cast<uintptr_t>(p) & (align - 1))
        return set_error(AAEDN_EINVAL, "%s: %s must be %zu-byte aligned", fn, what, align);
    cudaPointerAttributes at;
    const cudaError_t e = cudaPointerGetAttributes(&at, p);
    if (e != cudaSuccess)
    {
        cudaGetLastError();
        return set_error(AAEDN_EINVAL, "%s: %s: cannot query pointer (%s)", fn, what, cudaGetErrorString(e));
    }
    if (at.type != cudaMemoryTypeDevice && at.type != cudaMemoryTypeManaged)
        return set_error(AAEDN_EINVAL, "%s: %s is not device memory", fn, what);
    int dev = 0;
    AAEDN_CUDA_TRY(cudaGetDevice(&dev));
    if (at.type == cudaMemoryTypeDevice && at.device != dev)
        return set_error(AAEDN_EINVAL, "%s: %s is on device %d, the current device is %d", fn, what, at.device, dev);
    return AAEDN_OK;
}

} // namespace aaedn_dev
