// One kernel launch with its attributes: programmatic dependent launch and a
// cluster size.
#pragma once

#include <cuda_runtime.h>

namespace cq {

template <class... P, class... A>
cudaError_t launch_clustered(void (*kernel)(P...), dim3 grid, dim3 block, size_t smem, cudaStream_t stream, bool pdl,
                             int cluster, const A&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  int n = 0;
  if (pdl) {
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n++].val.programmaticStreamSerializationAllowed = 1;
  }
  if (cluster > 1) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = cluster;
    attr[n].val.clusterDim.y = 1;
    attr[n++].val.clusterDim.z = 1;
  }
  cfg.attrs = attr;
  cfg.numAttrs = n;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

template <class... P, class... A>
cudaError_t launch(void (*kernel)(P...), dim3 grid, dim3 block, size_t smem, cudaStream_t stream, bool pdl,
                   const A&... args) {
  return launch_clustered(kernel, grid, block, smem, stream, pdl, 1, args...);
}

}  // namespace cq
