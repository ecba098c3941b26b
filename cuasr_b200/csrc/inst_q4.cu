// Plans and launches the products with 4-bit weights.
#include <algorithm>

#include "decode_launch.h"
#include "q4_launch.cuh"
namespace cuasr_b200 {
namespace {

struct Q4Plan {
  int warps = 0, parts = 0, slices = 1, panel_steps = 0, grid = 0, sum_bytes = 0, smem = 0;
};
// What the shape of X makes of a block.
struct Q4Shape {
  int columns, column_tiles, rows, stage_bytes;      // rows: weight rows of a worker
};

// Shared memory of a block: stages, sums, X of a panel and what is read behind it (X is read eight columns at a time).
void fit(Q4Plan* plan, int slice_steps, const Q4Shape& s) {
  plan->sum_bytes = plan->warps / plan->parts * std::max(plan->parts - 1, 1) * s.column_tiles * 8 * (s.rows + kQ4SumPad) * 4;
  const int fixed = plan->sum_bytes + s.column_tiles * 8 * 64, all_stages = kQ4Stages * plan->warps * s.stage_bytes;
  const int per_step = 512 * s.columns, room = kQ4SmemPerBlock - fixed;
  int panel = slice_steps;
  if (panel > (room - all_stages) / per_step) panel = (room - all_stages) / per_step / plan->parts * plan->parts;
  plan->panel_steps = panel;
  plan->smem = fixed + panel * per_step + all_stages;
}

// clusters[i]: clusters of 2^i blocks that the device runs at a time.
Q4Plan plan_q4(int units, int steps, int passes, const Q4Shape& shape, const int (&clusters)[kQ4SliceChoices]) {
  Q4Plan best;
  double best_cost = 0;
  for (int warps = 16; warps >= (shape.column_tiles == 1 ? 8 : 16); warps /= 2)
    for (int parts = 1; parts <= 8; parts *= 2)
      for (int i = 0; i < kQ4SliceChoices && (i == 0 || 1 << i <= steps); ++i) {
        const int s = 1 << i;
        Q4Plan plan;
        plan.warps = warps;
        plan.parts = parts;
        plan.slices = s;
        const int workers = warps / parts, slice_steps = (steps + s - 1) / s;
        fit(&plan, slice_steps, shape);
        if (plan.panel_steps <= 0) continue;
        const int blocks = std::max(1, std::min((units + workers - 1) / workers, clusters[i]));
        const double rounds = static_cast<double>(((units + workers - 1) / workers + blocks - 1) / blocks) * passes;
        // In microseconds, from measurements between 1024 x 1024 and 128000 x 4096: a warp's step with all warps at it 1.7 (1.4 where
        // they are eight, 2 for 32 columns), a worker's sums 1.3, a cluster's 2 more; X laid out by a block 0.5 for a step of all its
        // columns' warps.  Every plan was timed for 24 shapes; the chosen one was the best or within 4 % of it for each.  (In
        // graphs.  One row, 14336 x 4096: 12.4 with four parts of 16 warps, 12.7 with two of two slices.  Eight rows, 128000 x 4096: 57 with
        // one part, 60 with two, 70 with eight.  Sixteen: 90 with one part, 89 with two, 100 with four.  Thirty-two rows, 8192 x 8192: 32 with
        // four slices of one part, 37 with two of two, 49 with four parts.)
        const double step = shape.column_tiles == 4 ? 2.0 : warps == 16 ? 1.7 : 1.4;
        const double restaged = plan.panel_steps < slice_steps ? rounds : passes;
        const double cost = rounds * ((slice_steps + parts - 1) / parts * step + (parts > 1 ? 1.3 : 1.0) + (s > 1 ? 2.0 : 0.0)) +
                            restaged * slice_steps * shape.columns * 0.5 / warps;
        plan.grid = blocks * s;
        // equal plans: the one on more SMs (32 rows, 500 x 1500, one slice: 9.3 us with eight parts, 11.6 with two, when it was chosen)
        if (best.smem == 0 || cost < best_cost || (cost == best_cost && plan.grid > best.grid)) {
          best_cost = cost;
          best = plan;
        }
      }
  return best;
}

// A cluster lies within one of the device's groups of SMs, whose sizes its multiple need not divide: of 148 SMs 132 are in
// clusters of four at a time.  One cluster more than that runs behind all others (128000 x 4096, 32 rows: 380 us with 37).
cudaError_t count_clusters(int (&clusters)[kQ4SliceChoices], int sms) {
  static std::atomic<uint64_t> known[64];          // by device: 16 bits for each size
  static_assert(kQ4SliceChoices <= 4, "16 bits each");
  int dev = 0;
  cudaError_t err = cudaGetDevice(&dev);
  if (err != cudaSuccess) return err;
  uint64_t packed = known[dev & 63].load(std::memory_order_relaxed);
  if (packed == 0) {
    for (int i = 0; i < kQ4SliceChoices; ++i) {
      int n = sms;
      if (i > 0 && (err = q4_active_clusters(1 << i, &n)) != cudaSuccess) return err;
      packed |= static_cast<uint64_t>(std::max(1, std::min(n, 0xFFFF))) << (16 * i);
    }
    known[dev & 63].store(packed, std::memory_order_relaxed);
  }
  for (int i = 0; i < kQ4SliceChoices; ++i) clusters[i] = static_cast<int>(packed >> (16 * i) & 0xFFFF);
  return cudaSuccess;
}

// Weight rows as bytes: boxes of a worker's rows by the 64 bytes of half a step; zeros outside.
bool weight_map(CUtensorMap* map, const cuasr_b200_q4_args_t& a, int rows) {
  using Encode = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                              const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
  static const Encode encode = [] {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) != cudaSuccess || q != cudaDriverEntryPointSuccess) f = nullptr;
    return reinterpret_cast<Encode>(f);
  }();
  if (encode == nullptr || reinterpret_cast<uintptr_t>(a.W) % 16 != 0 || a.ldw % 16 != 0 || a.ldw >= (1LL << 40)) return false;
  const cuuint64_t dims[2] = {static_cast<cuuint64_t>((static_cast<int64_t>(a.k) + 1) / 2), static_cast<cuuint64_t>(a.n)};
  const cuuint64_t strides[1] = {static_cast<cuuint64_t>(a.ldw)};
  const cuuint32_t box[2] = {kQ4Step / 4, static_cast<cuuint32_t>(rows)}, ones[2] = {1, 1};
  return encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<uint8_t*>(a.W), dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
                CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

}  // namespace

// Passes over the weights, each with up to 32 columns of X: as many rows, or ten of 32 bits.
static int q4_passes(const cuasr_b200_q4_args_t& a) { return (a.m - 1) / (a.dtype_x == CUASR_F32 ? 10 : 32) + 1; }

bool q4_fits(const cuasr_b200_q4_args_t& a) {
  // row and step numbers stay 32-bit up to a grid's stride behind the last
  return a.n <= 0x7FFE0000 && a.k <= 0x7FFE0000 && q4_passes(a) <= 65535;
}

cudaError_t launch_q4(const cuasr_b200_q4_args_t& a, const DeviceInfo& dev, int* launches) {
  Q4Params p = {};
  p.X = a.X; p.ldx = a.ldx; p.W = a.W; p.ldw = a.ldw; p.scales = a.scales; p.ld_scales = a.ld_scales;
  p.zeros = a.zeros; p.ld_zeros = a.ld_zeros; p.Y = a.Y; p.ldy = a.ldy;
  p.m = a.m; p.n = a.n; p.k = a.k; p.group = a.group;
  p.groups = static_cast<int>((static_cast<long long>(a.k) + a.group - 1) / a.group);
  p.group_shift = -1;
  for (int b = 5; b < 31; ++b)
    if (a.group == 1 << b) p.group_shift = b;
  p.type_x = a.dtype_x; p.type_y = a.dtype_y; p.type_scale = a.dtype_scale;
  p.status = dev.status;
  const int parts = a.dtype_x == CUASR_F32 ? 3 : 1, passes = q4_passes(a);
  p.rows = (a.m - 1) / passes + 1;
  const int columns = p.rows * parts, nt = columns <= 8 ? 1 : columns <= 16 ? 2 : 4;
  const size_t es = a.dtype_x == CUASR_F32 ? 4 : 2;
  p.x_vectors = reinterpret_cast<uintptr_t>(a.X) % 16 == 0 && (a.ldx * es % 16 == 0 || a.m == 1);
  const int lw = a.group % 128 == 0 || a.group >= a.k ? 4 : a.group % 64 == 0 ? 2 : 1;
  const int steps = (a.k + kQ4Step - 1) / kQ4Step;
  CUtensorMap map = {};
  const int tiles = nt == 1 ? 2 : 1;
  const bool tma = weight_map(&map, a, 16 * tiles);
  const Q4Shape shape = {columns, nt, 16 * tiles, (tma ? kQ4Stage<true, 1> : kQ4Stage<false, 1>) * tiles};
  p.units = (a.n - 1) / shape.rows + 1;
  int clusters[kQ4SliceChoices];
  cudaError_t err = count_clusters(clusters, dev.sms);
  if (err != cudaSuccess) return err;
  const Q4Plan plan = plan_q4(p.units, steps, passes, shape, clusters);
  if (plan.smem == 0) return cudaErrorInvalidValue;      // no launch fits: never for one block per SM and one slice
  p.parts = plan.parts; p.slices = plan.slices; p.panel_steps = plan.panel_steps; p.sum_bytes = plan.sum_bytes;
  const Q4Launch l = {plan.grid, passes, plan.smem, static_cast<cudaStream_t>(a.stream)};
  err = nt == 4            ? launch_q4_columns<4, 1, 16>(lw, tma, map, p, l)
        : nt == 2          ? launch_q4_columns<2, 1, 16>(lw, tma, map, p, l)
        : plan.warps == 16 ? launch_q4_columns<1, 2, 16>(lw, tma, map, p, l)
                           : launch_q4_columns<1, 2, 8>(lw, tma, map, p, l);
  if (err == cudaSuccess) ++*launches;
  return err;
}

}  // namespace cuasr_b200
