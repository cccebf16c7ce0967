// Launches whose blocks may be set up while the previous kernel of the stream
// finishes (programmatic dependent launch): takes the launch out of the path of
// a chain of short kernels.  The kernel calls after_previous_kernel() before it
// touches memory: it returns when the kernels before it have finished and their
// writes are visible, as at an ordinary launch.
#pragma once
#include <cuda_runtime.h>

namespace bw {

__device__ __forceinline__ void after_previous_kernel() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
// The next kernel's blocks may be set up from here on, as far as there is room.
__device__ __forceinline__ void let_next_kernel_start() { asm volatile("griddepcontrol.launch_dependents;"); }

template <typename... P, typename... A>
cudaError_t launch_early(void (*kernel)(P...), dim3 grid, dim3 block, size_t smem, cudaStream_t stream,
                         const A&... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

}  // namespace bw
