// Products with 4-bit weights, 8 columns at a time, 16 warps to a block.
#include "q4_launch.cuh"
namespace cuasr_b200 {
template cudaError_t launch_q4_columns<1, 2, 16>(int, bool, const CUtensorMap&, const Q4Params&, const Q4Launch&);

cudaError_t q4_active_clusters(int slices, int* clusters) {
  static std::atomic<uint64_t> allowed{0};
  auto kernel = q4_kernel<true, 1, 2, 16, 4, true, false>;
  cudaError_t err = allow_shared_memory(reinterpret_cast<const void*>(kernel), kQ4SmemPerBlock, allowed);
  if (err != cudaSuccess) return err;
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3(static_cast<unsigned>(slices));
  config.blockDim = dim3(32 * 16);
  config.dynamicSmemBytes = kQ4SmemPerBlock;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = static_cast<unsigned>(slices);
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  config.attrs = attr;
  config.numAttrs = 1;
  return cudaOccupancyMaxActiveClusters(clusters, kernel, &config);
}
}  // namespace cuasr_b200
