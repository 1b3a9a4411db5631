// Launch with programmatic dependent launch: the kernel may be scheduled while its predecessor in the stream drains and
// waits for it with griddep_wait() (common.cuh).
#pragma once

#include <cuda_runtime.h>

#include <utility>

#include "launchers.h"
#include "once.h"

namespace qw {

// The device that launches and settings go to.
inline int current_device() {
  int device = 0;
  check_cuda(cudaGetDevice(&device), "current device");
  return device;
}

// In clusters of `cluster` consecutive blocks.
template <typename... KArgs, typename... Args>
void launch_pdl_clusters(void (*kernel)(KArgs...), dim3 grid, dim3 block, int cluster, size_t smem, cudaStream_t stream,
                         const char* what, Args&&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cluster;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  check_cuda(cudaLaunchKernelEx(&cfg, kernel, std::forward<Args>(args)...), what);
}

template <typename... KArgs, typename... Args>
void launch_pdl(void (*kernel)(KArgs...), dim3 grid, dim3 block, size_t smem, cudaStream_t stream, const char* what,
                Args&&... args) {
  launch_pdl_clusters(kernel, grid, block, 1, smem, stream, what, std::forward<Args>(args)...);
}

}  // namespace qw
