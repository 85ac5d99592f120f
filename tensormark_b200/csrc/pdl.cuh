// pdl.cuh — launches whose prologue overlaps the kernel before them in the stream (programmatic dependent launch).
#pragma once

#include <cuda_runtime.h>

#include "common.cuh"

namespace tmc {

// The kernel begins before the one in front of it has ended; it calls pdl_enter() before it touches memory.
template <typename... P, typename... A>
inline void launch_overlapped(void (*kernel)(P...), dim3 grid, dim3 block, size_t smem, cudaStream_t st, A... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid; cfg.blockDim = block; cfg.dynamicSmemBytes = smem; cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at; cfg.numAttrs = 1;
    cudaLaunchKernelEx(&cfg, kernel, P(args)...);
}
// The same with `units` clusters of cs CTAs each. cs is one that the device is known to hold.
template <typename... P, typename... A>
inline bool launch_units(void (*kernel)(P...), unsigned units, unsigned cs, unsigned threads, size_t smem, cudaStream_t st, A... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(units * cs); cfg.blockDim = dim3(threads); cfg.dynamicSmemBytes = smem; cfg.stream = st;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = cs; at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
    cfg.attrs = at; cfg.numAttrs = cs > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, kernel, P(args)...) == cudaSuccess || check_launch("launch");
}
__device__ __forceinline__ void pdl_enter() {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
}

}  // namespace tmc
