// Launches of the 8-bit operators that overlap their set-up with the end of the
// kernel before them in the stream (programmatic dependent launch): an operator of
// a few tokens takes about as long as a launch.  Every kernel launched here
// calls dependents_may_start(), so that its successor's CTAs may be placed
// beside its last ones, and wait_for_inputs() in every thread before it
// touches global memory: it returns when all earlier work of the stream is
// complete and visible, so nothing is read early, and a kernel cannot finish
// before its predecessors have.
#pragma once

#include <cuda_runtime.h>

#include <utility>

namespace llvq {

__device__ __forceinline__ void dependents_may_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_for_inputs() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// cluster: CTAs per cluster along x.
template <typename... Params, typename... Args>
cudaError_t launch_overlapped(void (*kernel)(Params...), dim3 grid, int threads, size_t smem, int cluster,
                              cudaStream_t stream, Args&&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3((unsigned)threads, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)cluster;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 0 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kernel, std::forward<Args>(args)...);
}

}  // namespace llvq
