// State tensors follow the back-pointers of a search: dst[s, j] = src[s, parent[s, j]].
#pragma once

#include "ptx.cuh"

namespace cuasr_b200 {

// States of one launch; the parameters for eight are an eighth as large, which is host time (a call that reorders eight states of
// 0.5 MB is over on the device in 3 us).
constexpr int kReorderFew = 8, kReorderStates = 64;
constexpr int kReorderThreads = 128;

// A state as the kernel walks it: per search, `vectors` vectors of (1 << log_width) bytes for every beam; vector c lies in
// segment c / segment_vectors, position (c % segment_vectors) / position_vectors.  Positions that follow one another
// without a gap are one long position (limit_bytes says how many of its bytes a used position takes).
struct ReorderState {
  const char* src;
  char* dst;
  long long src_batch, src_beam, src_segment, src_position;
  long long dst_batch, dst_beam, dst_segment, dst_position;
  unsigned long long vectors, segment_vectors, position_vectors;
  long long limit_bytes;       // > 0: ragged, positions in one run: bytes of a position
  int positions;
  unsigned int first_block, blocks_per_batch;
  unsigned char log_width, in_place, ragged, wide;   // wide: vector numbers pass 32 bits
};
template <int STATES>
struct ReorderParams {
  const int* parents; long long ld_parents;
  const int* lengths;
  unsigned int* status;
  int beams, keep, states;
  ReorderState state[STATES];
};

// A column is one vector of every kept row: the thread that has it reads all it needs of the column before it writes, so
// a search is reordered in place without a copy, and rows that stay where they are are neither read nor written.
template <typename V, int ROWS>
__device__ __forceinline__ void move_column(int keep, const char* src, char* dst, long long src_beam, long long dst_beam,
                                            const int* from) {
  for (int j0 = 0; j0 < keep; j0 += ROWS) {        // more than one round only where src and dst are apart
    V v[ROWS];
#pragma unroll
    for (int j = 0; j < ROWS; ++j)
      if (j0 + j < keep && from[j0 + j] >= 0) v[j] = *reinterpret_cast<const V*>(src + from[j0 + j] * src_beam);
#pragma unroll
    for (int j = 0; j < ROWS; ++j)
      if (j0 + j < keep && from[j0 + j] >= 0) *reinterpret_cast<V*>(dst + (j0 + j) * dst_beam) = v[j];
  }
}

template <int ROWS, int STATES>
__global__ void __launch_bounds__(kReorderThreads) reorder_kernel(const __grid_constant__ ReorderParams<STATES> p) {
  extern __shared__ int from[];
  grid_dependency_wait();
  grid_dependency_launch();
  int lo = 0, hi = p.states - 1;                     // the state this block belongs to
  while (lo < hi) {
    const int mid = (lo + hi + 1) / 2;
    if (p.state[mid].first_block <= blockIdx.x) lo = mid;
    else hi = mid - 1;
  }
  const ReorderState& s = p.state[lo];
  const unsigned int block = blockIdx.x - s.first_block;
  const unsigned int batch = block / s.blocks_per_batch;
  for (int j = threadIdx.x; j < p.keep; j += kReorderThreads) {
    int f = p.parents[batch * p.ld_parents + j];
    if (f >= p.beams) {
      report_device_error(p.status, kDeviceIndexOutOfRange);
      f = -1;
    }
    from[j] = s.in_place && f == j ? -1 : f;
  }
  const int used = s.ragged ? min(max(p.lengths[batch], 0), s.positions) : s.positions;
  __syncthreads();
  const unsigned long long c = static_cast<unsigned long long>(block % s.blocks_per_batch) * kReorderThreads + threadIdx.x;
  if (c >= s.vectors) return;
  unsigned long long segment, position, offset;
  if (s.wide) {
    segment = c / s.segment_vectors; offset = c % s.segment_vectors;
    position = offset / s.position_vectors; offset %= s.position_vectors;
  } else {
    const unsigned int sv = static_cast<unsigned int>(s.segment_vectors), pv = static_cast<unsigned int>(s.position_vectors);
    const unsigned int c32 = static_cast<unsigned int>(c), in_segment = c32 % sv;
    segment = c32 / sv; position = in_segment / pv; offset = in_segment % pv;
  }
  offset <<= s.log_width;
  if (s.ragged) {
    if (s.limit_bytes > 0 ? static_cast<long long>(offset) >= used * s.limit_bytes : static_cast<int>(position) >= used) return;
  }
  const char* src = s.src + batch * s.src_batch + static_cast<long long>(segment) * s.src_segment +
                    static_cast<long long>(position) * s.src_position + static_cast<long long>(offset);
  char* dst = s.dst + batch * s.dst_batch + static_cast<long long>(segment) * s.dst_segment +
              static_cast<long long>(position) * s.dst_position + static_cast<long long>(offset);
  switch (s.log_width) {
    case 4: move_column<uint4, ROWS>(p.keep, src, dst, s.src_beam, s.dst_beam, from); break;
    case 3: move_column<uint2, ROWS>(p.keep, src, dst, s.src_beam, s.dst_beam, from); break;
    case 2: move_column<unsigned int, ROWS>(p.keep, src, dst, s.src_beam, s.dst_beam, from); break;
    case 1: move_column<unsigned short, ROWS>(p.keep, src, dst, s.src_beam, s.dst_beam, from); break;
    default: move_column<unsigned char, ROWS>(p.keep, src, dst, s.src_beam, s.dst_beam, from); break;
  }
}

}  // namespace cuasr_b200
