// Kernel launches: more than 48 KB of shared memory, and one launch with its attributes: programmatic dependent launch and a
// cluster size.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>

namespace cq {

// A kernel's opt-in to large dynamic shared memory, once per device.
class SharedMemoryOptIn {
 public:
  cudaError_t ensure(const void* kernel, int bytes) {
    int device = 0;
    cudaError_t e = cudaGetDevice(&device);
    if (e != cudaSuccess) return e;
    const uint64_t bit = 1ull << (device & 63);
    if (done_.load(std::memory_order_acquire) & bit) return cudaSuccess;
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == cudaSuccess) done_.fetch_or(bit, std::memory_order_release);
    return e;
  }

 private:
  std::atomic<uint64_t> done_{0};
};

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
