// Launches of the decoding kernels.  A decoding step is a chain of short kernels on one stream, so each is launched while the one
// before it still runs (programmatic stream serialization): it lets the next one start at once and waits for the one before
// before it touches memory (weights may be prefetched to L2 earlier; the kernel that joins attention reads lengths earlier, and is
// let start only when they are there).  Every thread waits, so that a kernel's end means the end of all before it.
// What a kernel before it may have written is read with ordinary loads: the read-only path (__ldg, or a __restrict__ pointer to const)
// is for memory that nothing writes while the kernel lives, which begins before that wait, and its loads may be moved across the wait.
#pragma once

#include <cuda_runtime.h>

namespace mts {

__device__ __forceinline__ void let_next_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_for_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

template <typename... Params, typename... Args>
cudaError_t launch_chained(void (*kernel)(Params...), dim3 grid, int threads, size_t shared, int cluster, cudaStream_t stream, const Args&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(unsigned(threads));
  cfg.dynamicSmemBytes = shared;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = unsigned(cluster);
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 0 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kernel, Params(args)...);
}

}  // namespace mts
