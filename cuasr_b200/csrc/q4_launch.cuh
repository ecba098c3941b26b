// Launchers of q4_kernel; instantiated by the number of columns in the inst_q4_*.cu files so that they compile in parallel.
#pragma once

#include "decode_launch.h"
#include "q4_product.cuh"

namespace cuasr_b200 {

// a block has some 300 bytes of static shared memory and 1 KB that the driver keeps
constexpr int kQ4SmemPerSm = 228 * 1024, kQ4SmemPerBlock = kQ4SmemPerSm - 2048;

struct Q4Launch {
  int grid_x, grid_y, smem;
  cudaStream_t stream;
};

template <bool BF16, int NT, int RT, int WARPS, int LW, bool TMA, bool ZEROS>
cudaError_t launch_q4_kernel(const CUtensorMap& map, const Q4Params& p, const Q4Launch& l) {
  static std::atomic<uint64_t> allowed{0};
  auto kernel = q4_kernel<BF16, NT, RT, WARPS, LW, TMA, ZEROS>;
  const cudaError_t err = allow_shared_memory(reinterpret_cast<const void*>(kernel), kQ4SmemPerBlock, allowed);
  if (err != cudaSuccess) return err;
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3(static_cast<unsigned>(l.grid_x), static_cast<unsigned>(l.grid_y));
  config.blockDim = dim3(32 * WARPS);
  config.dynamicSmemBytes = static_cast<size_t>(l.smem);
  config.stream = l.stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = static_cast<unsigned>(p.slices);
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  config.attrs = attr;
  config.numAttrs = p.slices > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&config, kernel, map, p);
}

// Clusters of `slices` blocks, each with an SM to itself, that the device runs at a time (inst_q4_1_16.cu).
cudaError_t q4_active_clusters(int slices, int* clusters);

template <int NT, int RT, int WARPS>
cudaError_t launch_q4_columns(int lw, bool tma, const CUtensorMap& map, const Q4Params& p, const Q4Launch& l) {
  const bool zeros = p.zeros != nullptr, bf16 = p.type_x != CUASR_F16;
#define Q4_CASE(L, V, Z)                                                            \
  if (lw == L && tma == V && zeros == Z)                                            \
    return bf16 ? launch_q4_kernel<true, NT, RT, WARPS, L, V, Z>(map, p, l) : launch_q4_kernel<false, NT, RT, WARPS, L, V, Z>(map, p, l);
#define Q4_CASES(L) Q4_CASE(L, false, false) Q4_CASE(L, true, false) Q4_CASE(L, false, true) Q4_CASE(L, true, true)
  Q4_CASES(1) Q4_CASES(2) Q4_CASES(4)
#undef Q4_CASES
#undef Q4_CASE
  return cudaErrorInvalidValue;
}

extern template cudaError_t launch_q4_columns<1, 2, 16>(int, bool, const CUtensorMap&, const Q4Params&, const Q4Launch&);
extern template cudaError_t launch_q4_columns<1, 2, 8>(int, bool, const CUtensorMap&, const Q4Params&, const Q4Launch&);
extern template cudaError_t launch_q4_columns<2, 1, 16>(int, bool, const CUtensorMap&, const Q4Params&, const Q4Launch&);
extern template cudaError_t launch_q4_columns<4, 1, 16>(int, bool, const CUtensorMap&, const Q4Params&, const Q4Launch&);

}  // namespace cuasr_b200
