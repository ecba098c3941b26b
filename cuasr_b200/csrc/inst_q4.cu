// Launcher of the products with 4-bit weights.
#include "decode_launch.h"
#include "q4_product.cuh"
#include "srgemm_launch.h"
namespace cuasr_b200 {
template <typename TX, typename TY, typename TS>
static cudaError_t launch(const cuasr_b200_q4_args_t& a, int* launches) {
  Q4Params p = {a.X, a.ldx, a.W, a.ldw, a.scales, a.ld_scales, a.zeros, a.ld_zeros, a.Y, a.ldy, a.m, a.n, a.k, a.group,
                static_cast<int>((static_cast<long long>(a.k) + a.group - 1) / a.group)};
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3((a.n + 7) / 8, (a.m + 3) / 4);
  config.blockDim = dim3(256);
  config.stream = static_cast<cudaStream_t>(a.stream);
  *launches = 1;
  return cudaLaunchKernelEx(&config, q4_rows_kernel<TX, TY, TS>, p);
}
template <typename TX, typename TY>
static cudaError_t by_scale(const cuasr_b200_q4_args_t& a, int* launches) {
  if (a.dtype_scale == CUASR_F32) return launch<TX, TY, float>(a, launches);
  return a.dtype_scale == CUASR_F16 ? launch<TX, TY, __half>(a, launches) : launch<TX, TY, __nv_bfloat16>(a, launches);
}
template <typename TX>
static cudaError_t by_y(const cuasr_b200_q4_args_t& a, int* launches) {
  if (a.dtype_y == CUASR_F32) return by_scale<TX, float>(a, launches);
  return a.dtype_y == CUASR_F16 ? by_scale<TX, __half>(a, launches) : by_scale<TX, __nv_bfloat16>(a, launches);
}
cudaError_t launch_q4(const cuasr_b200_q4_args_t& a, const DeviceInfo&, int* launches) {
  if (a.dtype_x == CUASR_F32) return by_y<float>(a, launches);
  return a.dtype_x == CUASR_F16 ? by_y<__half>(a, launches) : by_y<__nv_bfloat16>(a, launches);
}
}  // namespace cuasr_b200
