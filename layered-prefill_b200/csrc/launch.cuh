// Kernel launch with programmatic dependent launch: the kernel may become resident before the previous
// kernel of the stream has finished, run its set-up (barrier init, TMEM allocation, descriptor prefetch)
// and then block in grid_dependency_wait() until that kernel's results are complete and visible.
// Every kernel launched this way calls grid_dependency_wait() before it reads or writes anything another
// kernel touches, so "previous kernel finished" stays transitive along the stream.
// One exception: w4_mma_kernel (w4_gemv.cu), as the down pass or behind quant_x_kernel, reads topk_ids and the codes before
// its wait. That is sound because the kernel in front of it, always one of the same call, lets it start only after its own wait
// (grid_dependency_launch() behind grid_dependency_wait() in every CTA): whatever wrote the ids and the codes has finished by
// then. What the kernel in front itself writes is read behind the wait. A kernel that lets its successor start first, as most
// here do, may not stand in front of one that reads early.
// MOE_B200_PDL=0 in the environment switches back to plain stream-ordered launches (debugging aid).
#pragma once

#include <cuda_runtime.h>

#include <cstdlib>
#include <utility>

namespace moe_b200 {

inline bool pdl_enabled() {
  static int v = -1;
  if (v < 0) {
    const char* e = getenv("MOE_B200_PDL");
    v = (e != nullptr && e[0] == '0') ? 0 : 1;
  }
  return v != 0;
}

template <typename... KArgs, typename... Args>
cudaError_t launch_pdl(void (*kernel)(KArgs...), dim3 grid, dim3 block, size_t smem, cudaStream_t stream,
                       Args&&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl_enabled() ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kernel, static_cast<KArgs>(std::forward<Args>(args))...);
}

// Same, with the grid grouped into thread-block clusters of `cluster_x` consecutive CTAs.
template <typename... KArgs, typename... Args>
cudaError_t launch_pdl_cluster(void (*kernel)(KArgs...), dim3 grid, dim3 block, size_t smem, cudaStream_t stream,
                               unsigned cluster_x, Args&&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = cluster_x;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl_enabled() ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kernel, static_cast<KArgs>(std::forward<Args>(args))...);
}

// Blocks until the previous kernel of the stream has completed (no-op for a plain launch).
__device__ __forceinline__ void grid_dependency_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
// Lets the next kernel of the stream start becoming resident.
__device__ __forceinline__ void grid_dependency_launch() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

}  // namespace moe_b200
