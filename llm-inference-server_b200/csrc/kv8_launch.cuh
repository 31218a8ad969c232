// Launches that overlap with their predecessor's end (programmatic dependent launch): the
// kernels of one attention call are short and each would otherwise pay the gap of a launch.
//
// Every kernel launched this way waits (pdl_wait) before it touches global memory, or, where
// what it reads was complete before its predecessor started, before it ends; so a kernel's
// completion still implies its predecessor's.  pdl_release lets the successor's blocks start
// where there is room.
#pragma once

#include <cuda_runtime.h>

namespace pa {

__device__ __forceinline__ void pdl_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void pdl_release() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

template <typename... P, typename... A>
static cudaError_t launch_pdl(void (*kern)(P...), dim3 grid, dim3 block, size_t smem, cudaStream_t stream, A... args) {
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kern, args...);
}

}  // namespace pa
