// One step of beam searches: the `keep` best of beams x vocab continuations, a max-plus step with back-pointers.
//
//   value(b, v) = (score[b] - log sum_u exp(logit[b, u])) + logit[b, v]
//
// Within a prefix the values order as its logits do, so one pass over the logits finds both the sum and the prefix's own
// `keep` best; the searches' best are then chosen among those.
#pragma once

#include "decode_types.cuh"

namespace cuasr_b200 {

constexpr int kBeamThreads = 256;
constexpr int kBeamItems = 16;                                  // logits of a thread per tile
constexpr int kBeamTile = kBeamThreads * kBeamItems;
constexpr int kBeamList = 1024;                                 // candidates kept between tiles before they are thinned out
constexpr int kBeamMergeTile = 4 * kBeamThreads;
constexpr int kBeamMergeList = 512;

struct BeamParams {
  const void* logits; long long batch_stride, beam_stride;
  const float* scores; long long ld_scores;
  const unsigned char* finished; long long ld_finished;
  float* out_scores; long long ld_out_scores;
  int* parents; long long ld_parents;
  int* tokens; long long ld_tokens;
  unsigned long long* part_keys;   // [batch * beams * parts][keep], best first, 0 behind the last
  double* part_sum;                // [batch * beams * parts]: sum of exp(logit - part_max)
  float* part_max;
  int batch, beams, vocab, keep, parts, end_token, normalise;
};

// Whole numbers that order as (logit, lower token first); 0 is no candidate.
__device__ __forceinline__ unsigned long long beam_key(float x, int token) {
  const unsigned int bits = __float_as_uint(x + 0.0f);           // one zero
  const unsigned int up = bits >> 31 ? ~bits : bits | 0x80000000u;
  return static_cast<unsigned long long>(up) << 32 | static_cast<unsigned int>(~token);
}
__device__ __forceinline__ float beam_key_logit(unsigned long long key) {
  const unsigned int up = static_cast<unsigned int>(key >> 32);
  return __uint_as_float(up >> 31 ? up & 0x7FFFFFFFu : ~up);
}
__device__ __forceinline__ int beam_key_token(unsigned long long key) { return static_cast<int>(~static_cast<unsigned int>(key)); }

// exp(d) for d <= 0: log2(e) in two parts, since one 32-bit factor would shift every term the same way and the sum by
// 1e-7 of itself.
__device__ __forceinline__ float exp_of(float d) {
  const float y = fmaf(d, 1.44269502162933349609375f, d * 1.92596299112661746887e-8f);
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(y));
  return r;
}

// The largest float below x (x finite or +infinity; -infinity stays).
__device__ __forceinline__ float float_below(float x) {
  if (x == 0.0f) return -__uint_as_float(1u);
  const unsigned int bits = __float_as_uint(x);
  if (bits == 0xFF800000u) return x;
  return __uint_as_float(bits >> 31 ? bits + 1 : bits - 1);
}

// A list of candidate keys in shared memory that `keep` survivors are chosen from.
struct BeamList {
  unsigned long long* keys;    // kBeamList + kBeamTile
  int* count;
};

// The keep-th largest of n distinct keys, found bit by bit.  All threads call it.
__device__ __forceinline__ unsigned long long kth_key(const unsigned long long* keys, int n, int keep, int* counter) {
  unsigned long long found = 0;
  for (int bit = 63; bit >= 0; --bit) {
    const unsigned long long probe = found | 1ull << bit;
    int c = 0;
    for (int i = threadIdx.x; i < n; i += kBeamThreads) c += keys[i] >= probe;
    c = __reduce_add_sync(0xFFFFFFFFu, c);
    if (threadIdx.x == 0) *counter = 0;
    __syncthreads();
    if (threadIdx.x % 32 == 0) atomicAdd(counter, c);
    __syncthreads();
    if (*counter >= keep) found = probe;
    __syncthreads();
  }
  return found;
}

// Leaves the `keep` largest of the list at its front, in no order; returns the smallest of them.
__device__ __forceinline__ unsigned long long thin_out(const BeamList& list, int keep, int* counter) {
  __syncthreads();
  const int n = *list.count;
  const unsigned long long least = kth_key(list.keys, n, keep, counter);
  constexpr int kMost = (kBeamList + kBeamTile + kBeamThreads - 1) / kBeamThreads;
  unsigned long long mine[kMost];
#pragma unroll
  for (int i = 0; i < kMost; ++i) {
    const int at = i * kBeamThreads + threadIdx.x;
    mine[i] = at < n ? list.keys[at] : 0;
  }
  __syncthreads();
  if (threadIdx.x == 0) *list.count = 0;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kMost; ++i)
    if (mine[i] != 0 && mine[i] >= least) list.keys[atomicAdd(list.count, 1)] = mine[i];
  __syncthreads();
  return least;
}

template <typename T>
__global__ void __launch_bounds__(kBeamThreads) beam_part_kernel(const BeamParams p) {
  extern __shared__ unsigned long long beam_smem[];
  __shared__ int count, counter;
  __shared__ float maxima[kBeamThreads];
  __shared__ double sums[kBeamThreads / 32];
  __shared__ float limit;
  constexpr int V = Vec16<T>::count, U = kBeamItems / V;
  const int tid = threadIdx.x;
  const long long row = blockIdx.x / p.parts;
  const int part = blockIdx.x % p.parts;
  const int batch = static_cast<int>(row / p.beams), beam = static_cast<int>(row % p.beams);
  grid_dependency_wait();
  grid_dependency_launch();
  if (p.finished != nullptr && p.finished[batch * p.ld_finished + beam] != 0) return;

  BeamList list = {beam_smem, &count};
  if (tid == 0) count = 0;
  const T* x = static_cast<const T*>(p.logits) + batch * p.batch_stride + beam * p.beam_stride;
  // the row: up to V - 1 logits before the first 16-byte boundary, whole vectors, up to V - 1 logits behind them
  const int head = min(p.vocab, static_cast<int>((16 - reinterpret_cast<uintptr_t>(x) % 16) % 16 / sizeof(T)));
  const int vectors = (p.vocab - head) / V, tail = p.vocab - head - vectors * V;
  const int v_begin = static_cast<int>(static_cast<long long>(vectors) * part / p.parts);
  const int v_end = static_cast<int>(static_cast<long long>(vectors) * (part + 1) / p.parts);
  const uint4* xv = reinterpret_cast<const uint4*>(x + head);

  float m = -INFINITY, sum = 0.0f, above = -INFINITY;    // this thread's maximum and sum; candidates are above `above`
  __syncthreads();

  // the few logits outside of whole vectors, one to a thread: those in front first, those behind last, so that of equal
  // logits the ones met later always have the higher token
  auto take_one = [&](int at) {
    const float value = to_float(x[at]);
    if (value > above) list.keys[atomicAdd(&count, 1)] = beam_key(value, at);
    const float m_new = fmaxf(m, value), ref = m_new == -INFINITY ? 0.0f : m_new;
    sum = fmaf(sum, exp_of(m - ref), exp_of(value - ref));
    m = m_new;
  };
  if (part == 0 && tid < head) take_one(tid);
  for (int base = v_begin; base < v_end; base += kBeamThreads * U) {
    float v[U][V];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int at = base + u * kBeamThreads + tid;
      if (at < v_end) unpack16(__ldcs(xv + at), v[u], T());
      else {
#pragma unroll
        for (int e = 0; e < V; ++e) v[u][e] = -INFINITY;
      }
    }
    float top = -INFINITY;
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int e = 0; e < V; ++e) top = fmaxf(top, v[u][e]);
    if (p.normalise) {
      const float m_new = fmaxf(m, top), ref = m_new == -INFINITY ? 0.0f : m_new;
      float s = 0.0f;
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int e = 0; e < V; ++e) s += exp_of(v[u][e] - ref);
      sum = fmaf(sum, exp_of(m - ref), s);
      m = m_new;
    }
    if (base == v_begin) {
      // keep threads have a logit at or above the keep-th largest of the threads' maxima
      maxima[tid] = top;
      if (tid == 0) limit = -INFINITY;
      __syncthreads();
      int rank = 0;
#pragma unroll 8
      for (int i = 0; i < kBeamThreads; ++i) rank += maxima[i] > top || (maxima[i] == top && i < tid);
      if (rank == p.keep - 1) limit = float_below(top);
      __syncthreads();
      above = limit;
    }
    if (top > above) {
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int e = 0; e < V; ++e)
          if (v[u][e] > above)
            list.keys[atomicAdd(&count, 1)] = beam_key(v[u][e], head + (base + u * kBeamThreads + tid) * V + e);
    }
    __syncthreads();
    if (count > kBeamList) {
      // what follows lies further along the row: equal logits there lose
      above = beam_key_logit(thin_out(list, p.keep, &counter));
    }
    __syncthreads();
  }
  if (part == p.parts - 1 && tid < tail) take_one(p.vocab - tail + tid);
  __syncthreads();
  if (count > kBeamMergeList) thin_out(list, p.keep, &counter);
  __syncthreads();
  const int n = count;
  unsigned long long* out = p.part_keys + static_cast<long long>(blockIdx.x) * p.keep;
  for (int i = tid; i < n; i += kBeamThreads) {
    const unsigned long long key = list.keys[i];
    int rank = 0;
    for (int j = 0; j < n; ++j) rank += list.keys[j] > key;
    if (rank < p.keep) out[rank] = key;
  }
  for (int i = n + tid; i < p.keep; i += kBeamThreads) out[i] = 0;

  if (p.normalise) {
    maxima[tid] = m;
    __syncthreads();
    float all = -INFINITY;
    for (int i = tid % 32; i < kBeamThreads; i += 32) all = fmaxf(all, maxima[i]);
#pragma unroll
    for (int o = 16; o > 0; o /= 2) all = fmaxf(all, __shfl_xor_sync(0xFFFFFFFFu, all, o));
    // a thread without a logit above -infinity has a sum of 0, or NaN
    double s = m == -INFINITY ? static_cast<double>(sum) : static_cast<double>(sum) * exp(static_cast<double>(m) - static_cast<double>(all));
#pragma unroll
    for (int o = 16; o > 0; o /= 2) s += __shfl_xor_sync(0xFFFFFFFFu, s, o);
    if (tid % 32 == 0) sums[tid / 32] = s;
    __syncthreads();
    if (tid == 0) {
      for (int i = 1; i < kBeamThreads / 32; ++i) s += sums[i];
      p.part_max[blockIdx.x] = all;
      p.part_sum[blockIdx.x] = s;
    }
  }
}

// One block per search: log-sums of its prefixes, then the best of all parts' candidates.
struct BeamEntry {
  double value;
  unsigned long long key;
  int beam, pad;
};
__device__ __forceinline__ bool better(const BeamEntry& a, const BeamEntry& b) {
  if (a.value != b.value) return a.value > b.value;
  if (a.beam != b.beam) return a.beam < b.beam;
  return a.key > b.key;
}

__global__ void __launch_bounds__(kBeamThreads) beam_merge_kernel(const BeamParams p) {
  extern __shared__ unsigned long long beam_smem[];
  __shared__ int count;
  __shared__ double maxima[kBeamThreads];
  __shared__ double limit;
  double* base = reinterpret_cast<double*>(beam_smem);                     // [beams]: score, less the log-sum
  BeamEntry* list = reinterpret_cast<BeamEntry*>(base + p.beams + p.beams % 2);   // kBeamMergeList + kBeamMergeTile
  BeamEntry* best = list + kBeamMergeList + kBeamMergeTile;                // keep
  unsigned char* done = reinterpret_cast<unsigned char*>(best + p.keep);   // [beams]
  const int tid = threadIdx.x, batch = blockIdx.x;
  grid_dependency_wait();
  grid_dependency_launch();
  if (tid == 0) { count = 0; limit = -INFINITY; }
  for (int b = tid / 32; b < p.beams; b += kBeamThreads / 32) {
    const bool ended = p.finished != nullptr && p.finished[batch * p.ld_finished + b] != 0;
    double value = p.scores[batch * p.ld_scores + b];
    if (p.normalise && !ended) {
      const long long first = (static_cast<long long>(batch) * p.beams + b) * p.parts;
      float all = -INFINITY;
      for (int i = tid % 32; i < p.parts; i += 32) all = fmaxf(all, p.part_max[first + i]);
#pragma unroll
      for (int o = 16; o > 0; o /= 2) all = fmaxf(all, __shfl_xor_sync(0xFFFFFFFFu, all, o));
      double s = 0.0;
      for (int i = tid % 32; i < p.parts; i += 32) {
        const float m = p.part_max[first + i];
        s += m == -INFINITY ? p.part_sum[first + i] : p.part_sum[first + i] * exp(static_cast<double>(m) - static_cast<double>(all));
      }
#pragma unroll
      for (int o = 16; o > 0; o /= 2) s += __shfl_xor_sync(0xFFFFFFFFu, s, o);
      value -= (all == -INFINITY ? 0.0 : static_cast<double>(all)) + log(s);
    }
    if (tid % 32 == 0) { base[b] = value; done[b] = ended; }
  }
  __syncthreads();

  const int per_beam = p.parts * p.keep;
  const long long entries = static_cast<long long>(p.beams) * per_beam;
  const unsigned long long* keys = p.part_keys + static_cast<long long>(batch) * entries;
  double above = -INFINITY;
  bool at_least = false;                      // candidates are above `above`, or (at_least) at it too
  for (long long from = 0; from < entries; from += kBeamMergeTile) {
    BeamEntry e[4];
    double top = -INFINITY;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const long long at = from + u * kBeamThreads + tid;
      e[u].value = -INFINITY; e[u].key = 0; e[u].beam = 0; e[u].pad = 0;
      if (at < entries) {
        const int b = static_cast<int>(at / per_beam);
        e[u].beam = b;
        if (done[b]) {
          if (at % per_beam == 0) {
            e[u].value = base[b];
            e[u].key = static_cast<unsigned int>(~p.end_token);
          }
        } else {
          e[u].key = keys[at];
          if (e[u].key != 0) e[u].value = base[b] + static_cast<double>(beam_key_logit(e[u].key));
        }
        if (!(e[u].value > -INFINITY)) e[u].value = -INFINITY;      // NaN is no candidate
      }
      top = fmax(top, e[u].value);
    }
    if (from == 0) {
      maxima[tid] = top;
      __syncthreads();
      int rank = 0;
#pragma unroll 8
      for (int i = 0; i < kBeamThreads; ++i) rank += maxima[i] > top || (maxima[i] == top && i < tid);
      if (rank == p.keep - 1) limit = top;
      __syncthreads();
      above = limit;
      at_least = above > -INFINITY;
    }
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (e[u].value > above || (at_least && e[u].value == above)) list[atomicAdd(&count, 1)] = e[u];
    __syncthreads();
    const int n = count;
    const bool last = from + kBeamMergeTile >= entries;
    if (n > kBeamMergeList || last) {
      for (int i = tid; i < n; i += kBeamThreads) {
        const BeamEntry mine = list[i];
        int rank = 0;
        for (int j = 0; j < n; ++j) rank += better(list[j], mine);
        if (rank < p.keep) best[rank] = mine;
      }
      __syncthreads();
      const int kept = min(n, p.keep);
      if (!last) {
        for (int i = tid; i < kept; i += kBeamThreads) list[i] = best[i];
        if (tid == 0) count = kept;
        if (kept == p.keep) { above = best[kept - 1].value; at_least = true; }
      } else {
        for (int i = tid; i < p.keep; i += kBeamThreads) {
          const bool some = i < kept;
          p.out_scores[batch * p.ld_out_scores + i] = some ? static_cast<float>(best[i].value) : -INFINITY;
          p.parents[batch * p.ld_parents + i] = some ? best[i].beam : -1;
          p.tokens[batch * p.ld_tokens + i] = some ? beam_key_token(best[i].key) : -1;
        }
      }
    }
    __syncthreads();
  }
}

}  // namespace cuasr_b200
