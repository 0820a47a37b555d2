// Host side of thread-block clusters: how many run at one time.
#pragma once

#include <atomic>

#include "common.cuh"

namespace gdn2 {

constexpr int kMaxPortableCluster = 8, kMaxLargeCluster = 16;

struct ClusterMemo {
  std::atomic<int> n[64][kMaxLargeCluster];             // per device ordinal and size; 0 = not asked yet
};

// Clusters of more than 8 blocks have to be asked for, on every device
inline cudaError_t allow_large_clusters(const void* kernel) {
  return cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
}

// A cluster lies within a group of SMs, and what does not fill one up is lost (B200, one block an SM: 148, 74, 45, 33, 26, 22, 15
// and 15 clusters of 1 to 8 blocks, 7 of 12 and of 16; two: 296, 148, 93, 71, 56, 45, 37, 33, 21 and 14). Asked once per device, memo
// and size.
inline int active_clusters(ClusterMemo& memo, const void* kernel, int threads, size_t smem, int per_sm, int cl) {
  int dev = 0, n = 0;
  const bool kept = cudaGetDevice(&dev) == cudaSuccess && dev >= 0 && dev < 64;
  if (kept && (n = memo.n[dev][cl - 1].load()) > 0) return n;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = cl;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(cl);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (ensure_dynamic_smem(kernel, smem) != cudaSuccess || (cl > kMaxPortableCluster && allow_large_clusters(kernel) != cudaSuccess) ||
      cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess || n <= 0) {
    cudaGetLastError();                                  // not this call's failure: an estimate will do
    n = per_sm * device_sm_count() / cl;
    return n > 0 ? n : 1;
  }
  if (kept) memo.n[dev][cl - 1].store(n);
  return n;
}

}  // namespace gdn2
