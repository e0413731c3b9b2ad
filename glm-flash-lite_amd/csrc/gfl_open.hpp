// Kernels that use more LDS than a launch may take by default.
#pragma once
#include <hip/hip_runtime.h>

#include <atomic>

namespace gfl {

// Allows a kernel its LDS, once on each device (the attribute belongs to the device's copy of the kernel; `opened`: a bit for each).
static inline void gm_open(const void* kern, int lds, std::atomic<uint64_t>& opened)
{
    int dev = 0;
    if (hipGetDevice(&dev) != hipSuccess) return;   // the launch reports it
    const uint64_t bit = dev < 64 ? 1ull << dev : 0;
    if (bit && (opened.load(std::memory_order_relaxed) & bit)) return;
    if (hipFuncSetAttribute(kern, hipFuncAttributeMaxDynamicSharedMemorySize, lds) == hipSuccess) opened.fetch_or(bit);
}

}  // namespace gfl
