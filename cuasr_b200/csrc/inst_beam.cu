// Launcher of the beam steps.
#include <algorithm>

#include "beam_step.cuh"
#include "decode_launch.h"
#include "srgemm_launch.h"
namespace cuasr_b200 {

// As many blocks as the SMs hold at a time, where every part still has a tile and the candidates fit into the merge's shared
// memory.  (32 searches of four prefixes over 128000 logits of 16 bits: 23 us with eight
// parts, 25 with six, 29 with three, when it was chosen; 18.5 with eight now.)
int beam_parts(const cuasr_b200_beam_args_t& a) {
  const long long rows = static_cast<long long>(a.batch) * a.beams;
  const int tile = kBeamThreads * kBeamVectors * (a.dtype == CUASR_F32 ? 4 : 8);
  const long long fill = kBeamBlocks * 148 / rows, tiles = (static_cast<long long>(a.vocab) + tile - 1) / tile;
  const long long room = std::min(kBeamMergeMost / (a.beams * a.keep), kMergeThreads / a.beams);
  return static_cast<int>(std::max(1LL, std::min({fill, tiles, room, 32LL})));
}

size_t beam_workspace_bytes(const cuasr_b200_beam_args_t& a) {
  const size_t parts = static_cast<size_t>(a.batch) * a.beams * beam_parts(a);
  return parts * (a.keep * sizeof(unsigned long long) + sizeof(double) + sizeof(float));
}

template <typename T, bool NORMALISE>
static cudaError_t launch_part(const BeamParams& p, cudaStream_t stream) {
  static std::atomic<uint64_t> allowed{0};
  constexpr int smem = kBeamStages * kBeamTileBytes;
  auto kernel = beam_part_kernel<T, NORMALISE>;
  const cudaError_t err = allow_shared_memory(reinterpret_cast<const void*>(kernel), smem, allowed);
  if (err != cudaSuccess) return err;
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3(static_cast<unsigned>(p.batch) * static_cast<unsigned>(p.beams), static_cast<unsigned>(p.parts));
  config.blockDim = dim3(kBeamThreads);
  config.dynamicSmemBytes = smem;
  config.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  config.attrs = attr;
  config.numAttrs = 1;
  return cudaLaunchKernelEx(&config, kernel, p);
}
template <typename T>
static cudaError_t launch_parts(const BeamParams& p, cudaStream_t stream) {
  return p.normalise ? launch_part<T, true>(p, stream) : launch_part<T, false>(p, stream);
}

cudaError_t launch_beam(const cuasr_b200_beam_args_t& a, const DeviceInfo& dev, int* launches) {
  BeamParams p = {};
  p.logits = a.logits; p.batch_stride = a.batch_stride; p.beam_stride = a.beam_stride;
  p.scores = a.scores; p.ld_scores = a.ld_scores;
  p.finished = a.finished; p.ld_finished = a.ld_finished;
  p.out_scores = a.out_scores; p.ld_out_scores = a.ld_out_scores;
  p.parents = a.parents; p.ld_parents = a.ld_parents;
  p.tokens = a.tokens; p.ld_tokens = a.ld_tokens;
  p.batch = a.batch; p.beams = a.beams; p.vocab = a.vocab; p.keep = a.keep;
  p.parts = beam_parts(a); p.end_token = a.end_token; p.normalise = a.normalise != 0;
  p.status = dev.status;
  const size_t parts = static_cast<size_t>(a.batch) * a.beams * p.parts;
  p.part_keys = static_cast<unsigned long long*>(a.workspace);
  p.part_sum = reinterpret_cast<double*>(p.part_keys + parts * a.keep);
  p.part_max = reinterpret_cast<float*>(p.part_sum + parts);
  cudaStream_t stream = static_cast<cudaStream_t>(a.stream);
  const int per_vector = a.dtype == CUASR_F32 ? 4 : 8;
  p.chunk = (a.vocab / per_vector + p.parts - 1) / p.parts;
  cudaError_t err = a.dtype == CUASR_F32   ? launch_parts<float>(p, stream)
                    : a.dtype == CUASR_F16 ? launch_parts<__half>(p, stream)
                                           : launch_parts<__nv_bfloat16>(p, stream);
  if (err != cudaSuccess) return err;
  ++*launches;
  const int lists = a.beams * p.parts, entries = lists * a.keep;
  const bool merged = entries <= kBeamMergeMost && lists <= kMergeThreads;
  const size_t smem = (merged ? entries * sizeof(BeamMerged) : 0) + beam_merge_scratch(a.keep) + a.beams * (sizeof(double) + 1) + lists;
  if (smem > 47 * 1024) {             // the kernel has a few bytes of its own
    static std::atomic<uint64_t> allowed{0};
    err = allow_shared_memory(reinterpret_cast<const void*>(beam_merge_kernel), 200 * 1024, allowed);
    if (err != cudaSuccess) return err;
  }
  err = launch_overlapped(beam_merge_kernel, a.batch, kMergeThreads, static_cast<int>(smem), 1, stream, p);
  if (err == cudaSuccess) ++*launches;
  return err;
}

}  // namespace cuasr_b200
