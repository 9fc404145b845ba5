// A kernel's opt-in to more shared memory than 48 KB.
#pragma once
#include <cuda_runtime.h>

#include <atomic>
#include <mutex>

// The attribute belongs to a kernel on the current device and holds for whoever launches it next, and host threads call at once: it is only ever
// raised, under a lock, so that no thread lowers it between another one's opt-in and launch.  A size that was allowed before costs a look at
// `size` (the call itself costs the host 0.4 us).
struct LlbSharedMemory {
    std::atomic<int> size[64] = {};
    std::mutex raising;
    template <typename Kernel> cudaError_t allow(Kernel* kernel, size_t bytes) {
        int device = 0;
        cudaError_t e = cudaGetDevice(&device);
        if (e != cudaSuccess) return e;
        if (device < 0 || device >= 64) return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
        if (size[device].load(std::memory_order_acquire) >= (int)bytes) return cudaSuccess;
        std::lock_guard<std::mutex> one_by_one(raising);
        if (size[device].load(std::memory_order_relaxed) >= (int)bytes) return cudaSuccess;
        e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
        if (e == cudaSuccess) size[device].store((int)bytes, std::memory_order_release);
        return e;
    }
};
