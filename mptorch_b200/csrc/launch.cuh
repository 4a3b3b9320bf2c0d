// Kernels of one call that follow one another: the second may start while the first still runs, does what does not depend on it, and
// then waits for it (programmatic dependent launch).
#pragma once
#include <atomic>

#include "common.cuh"

namespace mpt {

// In the first kernel: the next one may start.  In the second: everything the first one wrote is visible from here on.
__device__ __forceinline__ void next_may_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_for_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// Allows `Kern` up to `bytes` of dynamic shared memory, asked of the runtime once for each device.
template <auto Kern>
bool allow_shared(int bytes) {
    static std::atomic<uint64_t> asked{0};
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return false;
    const uint64_t bit = dev < 64 ? (uint64_t)1 << dev : 0;       // (devices behind the 64th are asked each time)
    if (asked.load(std::memory_order_relaxed) & bit) return true;
    if (cudaFuncSetAttribute(Kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess) return false;
    asked.fetch_or(bit, std::memory_order_relaxed);
    return true;
}

// Launches `kern` so that it may start before the kernel launched just before it on the stream is done.
template <typename... P, typename... A>
cudaError_t launch_after(void (*kern)(P...), dim3 grid, dim3 block, size_t smem, cudaStream_t st, A&&... args) {
    cudaLaunchConfig_t c{};
    c.gridDim = grid;
    c.blockDim = block;
    c.dynamicSmemBytes = smem;
    c.stream = st;
    cudaLaunchAttribute a{};
    a.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    a.val.programmaticStreamSerializationAllowed = 1;
    c.attrs = &a;
    c.numAttrs = 1;
    return cudaLaunchKernelEx(&c, kern, static_cast<P>(args)...);
}

}  // namespace mpt
