// Kernels that start while the one before them in their stream still runs.
// Such a kernel may read what no kernel writes (a layer's weights) at once; all
// else, and every write, comes behind after_kernel_before(). Every block
// passes it, so a kernel that has ended means that those before it have.
#pragma once

#include <cuda_runtime.h>

#include <utility>

namespace trit {

__device__ __forceinline__ void after_kernel_before() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
// Lets the next such kernel start as this one's blocks, once all have begun, leave room.
__device__ __forceinline__ void let_next_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// Launches such a kernel, in clusters of `cluster` blocks.
template <class... P, class... A>
cudaError_t launch_early(void (*kernel)(P...), dim3 grid, dim3 block, size_t smem, cudaStream_t s, unsigned cluster,
                         A&&... args) {
  cudaLaunchConfig_t config{};
  config.gridDim = grid;
  config.blockDim = block;
  config.dynamicSmemBytes = smem;
  config.stream = s;
  cudaLaunchAttribute attrs[2] = {};
  attrs[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attrs[0].val.programmaticStreamSerializationAllowed = 1;
  attrs[1].id = cudaLaunchAttributeClusterDimension;
  attrs[1].val.clusterDim.x = cluster;
  attrs[1].val.clusterDim.y = attrs[1].val.clusterDim.z = 1;
  config.attrs = attrs;
  config.numAttrs = cluster > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&config, kernel, std::forward<A>(args)...);
}

}  // namespace trit
