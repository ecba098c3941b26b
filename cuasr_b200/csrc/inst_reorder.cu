// Launcher of the reordering of states.
#include <algorithm>

#include "decode_launch.h"
#include "reorder.cuh"
#include "srgemm_launch.h"
namespace cuasr_b200 {
namespace {

// The widest vector (at most 16 bytes) that divides every number given.
int log_width_of(std::initializer_list<unsigned long long> numbers) {
  unsigned long long all = 16;
  for (unsigned long long v : numbers) all |= v;
  int log_width = 0;
  while (log_width < 4 && (all >> log_width & 1) == 0) ++log_width;
  return log_width;
}

// Dimensions that follow one another without a gap on both sides become one; false where a number passes its field.
bool plan_state(const cuasr_b200_state_t& s, const cuasr_b200_reorder_args_t& a, ReorderState* out) {
  ReorderState r = {};
  r.src = static_cast<const char*>(s.src); r.dst = static_cast<char*>(s.dst);
  r.src_batch = s.src_batch; r.src_beam = s.src_beam; r.src_segment = s.src_segment; r.src_position = s.src_position;
  r.dst_batch = s.dst_batch; r.dst_beam = s.dst_beam; r.dst_segment = s.dst_segment; r.dst_position = s.dst_position;
  r.in_place = s.src == s.dst && s.src_batch == s.dst_batch && s.src_beam == s.dst_beam && s.src_segment == s.dst_segment &&
               s.src_position == s.dst_position;
  r.ragged = s.ragged != 0;
  r.positions = s.positions;
  long long segments = s.segments, positions = s.positions, bytes = s.bytes;
  if (positions == 1 || (s.src_position == bytes && s.dst_position == bytes)) {
    if (r.ragged) r.limit_bytes = bytes;
    bytes *= positions;
    positions = 1;
    r.src_position = r.dst_position = 0;
    if (!r.ragged && segments > 1 && s.src_segment == bytes && s.dst_segment == bytes) {
      bytes *= segments;
      segments = 1;
    }
  }
  if (segments == 1) r.src_segment = r.dst_segment = 0;
  if (a.batch == 1) r.src_batch = r.dst_batch = 0;
  if (a.beams == 1) r.src_beam = 0;
  if (a.keep == 1) r.dst_beam = 0;
  const int w = log_width_of({reinterpret_cast<unsigned long long>(s.src), reinterpret_cast<unsigned long long>(s.dst),
                              (unsigned long long)r.src_batch, (unsigned long long)r.src_beam, (unsigned long long)r.src_segment,
                              (unsigned long long)r.src_position, (unsigned long long)r.dst_batch, (unsigned long long)r.dst_beam,
                              (unsigned long long)r.dst_segment, (unsigned long long)r.dst_position, (unsigned long long)bytes,
                              (unsigned long long)r.limit_bytes});
  r.log_width = static_cast<unsigned char>(w);
  r.position_vectors = static_cast<unsigned long long>(bytes) >> w;
  r.segment_vectors = r.position_vectors * positions;
  r.vectors = r.segment_vectors * segments;
  r.wide = r.vectors > 0xFFFFFFFFull;
  const unsigned long long blocks = (r.vectors + kReorderThreads - 1) / kReorderThreads;
  if (blocks * a.batch > 0x7FFFFFFFull) return false;
  r.blocks_per_batch = static_cast<unsigned int>(blocks);
  *out = r;
  return true;
}

template <int STATES>
cudaError_t launch_some(const ReorderParams<STATES>& p, unsigned int grid, cudaStream_t stream) {
  const int smem = p.keep * static_cast<int>(sizeof(int));
  auto kernel = p.keep <= 4    ? reorder_kernel<4, STATES>
                : p.keep <= 8  ? reorder_kernel<8, STATES>
                : p.keep <= 16 ? reorder_kernel<16, STATES>
                               : reorder_kernel<32, STATES>;
  return launch_overlapped(kernel, static_cast<int>(grid), kReorderThreads, smem, 1, stream, p);
}

template <int STATES>
cudaError_t launch_states(const cuasr_b200_reorder_args_t& a, const DeviceInfo& dev, int* launches) {
  ReorderParams<STATES> p;         // states behind the last are not looked at
  p.parents = a.parents; p.ld_parents = a.ld_parents; p.lengths = a.lengths; p.status = dev.status;
  p.beams = a.beams; p.keep = a.keep; p.states = 0;
  unsigned long long grid = 0;
  for (int i = 0; i < a.n_states; ++i) {
    ReorderState r;
    if (!plan_state(a.states[i], a, &r)) return cudaErrorInvalidValue;     // reorder_fits() was asked before
    const unsigned long long blocks = static_cast<unsigned long long>(r.blocks_per_batch) * a.batch;
    if (p.states == STATES || grid + blocks > 0x7FFFFFFFull) {
      const cudaError_t err = launch_some(p, static_cast<unsigned int>(grid), static_cast<cudaStream_t>(a.stream));
      if (err != cudaSuccess) return err;
      ++*launches;
      p.states = 0;
      grid = 0;
    }
    r.first_block = static_cast<unsigned int>(grid);
    p.state[p.states++] = r;
    grid += blocks;
  }
  const cudaError_t err = launch_some(p, static_cast<unsigned int>(grid), static_cast<cudaStream_t>(a.stream));
  if (err == cudaSuccess) ++*launches;
  return err;
}

}  // namespace

bool reorder_fits(const cuasr_b200_reorder_args_t& a) {
  ReorderState r;
  for (int i = 0; i < a.n_states; ++i)
    if (!plan_state(a.states[i], a, &r)) return false;
  return true;
}

cudaError_t launch_reorder(const cuasr_b200_reorder_args_t& a, const DeviceInfo& dev, int* launches) {
  return a.n_states <= kReorderFew ? launch_states<kReorderFew>(a, dev, launches) : launch_states<kReorderStates>(a, dev, launches);
}

}  // namespace cuasr_b200
