// Launcher of the beam steps.
#include <algorithm>

#include "beam_step.cuh"
#include "decode_launch.h"
#include "srgemm_launch.h"
namespace cuasr_b200 {

int beam_parts(const cuasr_b200_beam_args_t& a) {
  const long long rows = static_cast<long long>(a.batch) * a.beams;
  const long long wanted = (4 * 148 + rows - 1) / rows, most = (a.vocab + 2047) / 2048;
  return static_cast<int>(std::max(1LL, std::min(wanted, most)));
}

size_t beam_workspace_bytes(const cuasr_b200_beam_args_t& a) {
  const size_t parts = static_cast<size_t>(a.batch) * a.beams * beam_parts(a);
  return parts * (a.keep * sizeof(unsigned long long) + sizeof(double) + sizeof(float));
}

template <typename T>
static cudaError_t launch_parts(const BeamParams& p, int grid, cudaStream_t stream) {
  constexpr int smem = (kBeamList + kBeamTile) * sizeof(unsigned long long);
  static_assert(smem <= 48 * 1024, "more shared memory has to be asked for");
  return launch_overlapped(beam_part_kernel<T>, grid, kBeamThreads, smem, 1, stream, p);
}

cudaError_t launch_beam(const cuasr_b200_beam_args_t& a, const DeviceInfo&, int* launches) {
  BeamParams p = {};
  p.logits = a.logits; p.batch_stride = a.batch_stride; p.beam_stride = a.beam_stride;
  p.scores = a.scores; p.ld_scores = a.ld_scores;
  p.finished = a.finished; p.ld_finished = a.ld_finished;
  p.out_scores = a.out_scores; p.ld_out_scores = a.ld_out_scores;
  p.parents = a.parents; p.ld_parents = a.ld_parents;
  p.tokens = a.tokens; p.ld_tokens = a.ld_tokens;
  p.batch = a.batch; p.beams = a.beams; p.vocab = a.vocab; p.keep = a.keep;
  p.parts = beam_parts(a); p.end_token = a.end_token; p.normalise = a.normalise != 0;
  const size_t parts = static_cast<size_t>(a.batch) * a.beams * p.parts;
  p.part_keys = static_cast<unsigned long long*>(a.workspace);
  p.part_sum = reinterpret_cast<double*>(p.part_keys + parts * a.keep);
  p.part_max = reinterpret_cast<float*>(p.part_sum + parts);
  cudaStream_t stream = static_cast<cudaStream_t>(a.stream);
  const int grid = static_cast<int>(parts);
  cudaError_t err = a.dtype == CUASR_F32   ? launch_parts<float>(p, grid, stream)
                    : a.dtype == CUASR_F16 ? launch_parts<__half>(p, grid, stream)
                                           : launch_parts<__nv_bfloat16>(p, grid, stream);
  if (err != cudaSuccess) return err;
  ++*launches;
  const size_t smem = (a.beams + a.beams % 2) * sizeof(double) + (kBeamMergeList + kBeamMergeTile + a.keep) * sizeof(BeamEntry) + a.beams;
  static_assert(1024 * 9 + (kBeamMergeList + kBeamMergeTile + CUASR_B200_BEAM_MAX_KEEP) * sizeof(BeamEntry) <= 48 * 1024,
                "more shared memory has to be asked for");
  err = launch_overlapped(beam_merge_kernel, a.batch, kBeamThreads, static_cast<int>(smem), 1, stream, p);
  if (err == cudaSuccess) ++*launches;
  return err;
}

}  // namespace cuasr_b200
