// Kernels of one call that follow one another (programmatic dependent launch): the later one is launched, and does what needs
// nothing of the earlier one's, while the earlier one's last CTAs run.
#pragma once
#include <cuda_runtime.h>

namespace {

// in the earlier kernel: once all its CTAs have come here, those of the later one may take the places that are free
__device__ __forceinline__ void next_may_start() { asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory"); }
// in the later kernel, before its first access to memory: the earlier one has ended and its writes are visible
__device__ __forceinline__ void wait_for_previous() { asm volatile("griddepcontrol.wait;\n" ::: "memory"); }

template <typename... P, typename... A>
cudaError_t launch_next(void (*kernel)(P...), dim3 grid, dim3 block, size_t smem, cudaStream_t st, const A&... args)
{
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid, cfg.blockDim = block, cfg.dynamicSmemBytes = smem, cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at, cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}

}  // namespace
