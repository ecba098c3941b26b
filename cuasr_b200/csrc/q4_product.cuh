// Plus-times product of a few rows with weights in 4 bits.
#pragma once

#include "decode_types.cuh"

namespace cuasr_b200 {

struct Q4Params {
  const void* X; long long ldx;
  const unsigned char* W; long long ldw;
  const void* scales; long long ld_scales;
  const unsigned char* zeros; long long ld_zeros;
  void* Y; long long ldy;
  int m, n, k, group, groups;
};

// One warp per weight row and up to four rows of X; the lanes share each group's bytes.
template <typename TX, typename TY, typename TS>
__global__ void __launch_bounds__(256) q4_rows_kernel(const Q4Params p) {
  grid_dependency_wait();
  grid_dependency_launch();
  const int lane = threadIdx.x % 32;
  const long long j = static_cast<long long>(blockIdx.x) * 8 + threadIdx.x / 32;
  const int r0 = blockIdx.y * 4;
  if (j >= p.n) return;
  const unsigned char* w = p.W + j * p.ldw;
  const TX* x = static_cast<const TX*>(p.X) + r0 * p.ldx;
  float acc[4] = {};
  for (int g = 0; g < p.groups; ++g) {
    const float scale = to_float(static_cast<const TS*>(p.scales)[j * p.ld_scales + g]);
    const int zero = p.zeros == nullptr ? 8 : p.zeros[j * p.ld_zeros + g] & 15;
    const int k_end = min(p.k, (g + 1) * p.group);
    float part[4] = {};
    for (int k = g * p.group + 2 * lane; k < k_end; k += 64) {
      const int byte = w[k / 2];
      const float lo = static_cast<float>((byte & 15) - zero), hi = static_cast<float>((byte >> 4) - zero);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        if (r0 + r >= p.m) break;
        part[r] = fmaf(lo, to_float(x[r * p.ldx + k]), part[r]);
        if (k + 1 < k_end) part[r] = fmaf(hi, to_float(x[r * p.ldx + k + 1]), part[r]);
      }
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) acc[r] = fmaf(scale, part[r], acc[r]);
  }
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    float s = acc[r];
#pragma unroll
    for (int o = 16; o > 0; o /= 2) s += __shfl_xor_sync(0xFFFFFFFFu, s, o);
    if (lane == 0 && r0 + r < p.m) static_cast<TY*>(p.Y)[(r0 + r) * p.ldy + j] = from_float<TY>(s);
  }
}

}  // namespace cuasr_b200
