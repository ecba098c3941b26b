// One step of beam searches: the `keep` best of beams x vocab continuations, a max-plus step with back-pointers.
//
//   value(b, v) = (score[b] - log sum_u exp(logit[b, u])) + logit[b, v]
//
// Within a prefix the values order as its logits do, so one pass over the logits finds both the sum and the prefix's own
// `keep` best; the searches' best are then chosen among those.  The floor is the logits' bytes at the memory's rate, which
// leaves about eleven instructions of a lane for a 16-bit logit and twice as many for a 32-bit one; so exponentials are worked
// out in pairs, and a logit is otherwise only part of a maximum, which is compared with a bound that nearly all threads stay
// below.  The bound comes from the threads' own maxima and is taken again after 1, 2, 4, ... tiles; a row of 16 tiles then has
// about seven candidates for each that is kept, which every warp collects by itself and which are sorted once, at the row's end.
//
// Measured: 64 searches of 16 prefixes over 64000 32-bit logits 60 us, 4.4 TB/s; 32 searches of four over 128000 16-bit logits, a
// third of the prefixes ended, 18.5 us.  A block's later tiles pass at the memory's rate (2.3 thousand clocks with seven blocks to
// an SM); the first three take two to three times as long while the bound is low, and all blocks have theirs at the same time.
#pragma once

#include <cfloat>

#include "decode_types.cuh"

namespace cuasr_b200 {

constexpr int kBeamThreads = 128;
constexpr int kBeamVectors = 4;                                 // 16-byte vectors of a thread per tile
constexpr int kBeamTileBytes = kBeamThreads * kBeamVectors * 16;
constexpr int kBeamStages = 3;
constexpr int kBeamBlocks = 7;                                  // of an SM
constexpr int kBeamWarps = kBeamThreads / 32;
constexpr int kBeamSegment = 128;                               // candidates that a warp can hold after a tile ...
constexpr int kBeamStride = kBeamSegment + 8;                   // ... and the few logits behind the last
constexpr int kBeamCapacity = kBeamWarps * kBeamStride;
constexpr int kBeamRanked = kBeamThreads;                       // up to so many are sorted by comparing all with all
constexpr int kMergeThreads = 256;
constexpr int kBeamMergeMost = 8192;                            // candidates that are merged in shared memory

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
  int chunk;                       // vectors of a part
  unsigned int* status;
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

// exp(d) for d of at most kBeamLag: log2(e) in two parts, since one 32-bit factor would shift every term the same way and the sum by
// 1e-7 of itself.
__device__ __forceinline__ float exp_of(float d) {
  const float y = fmaf(d, 1.44269502162933349609375f, d * 1.92596299112661746887e-8f);
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(y));
  return r;
}

// A thread's sum of exp(logit - ref) is in 64 bits, to which a tile's is added, and `ref` is its maximum of some tile: it is taken
// anew, and the sum multiplied by a 32-bit exponential, only where the maximum has risen by more than kBeamLag above it, so the roundings of these
// do not add up however long the row is or slowly its logits rise.
constexpr float kBeamLag = 16.0f;

// ... of a pair.
__device__ __forceinline__ uint64_t exp_of_pair(uint64_t d) {
  const uint64_t y = fma2(d, pack2(1.44269502162933349609375f, 1.44269502162933349609375f),
                          mul2(d, pack2(1.92596299112661746887e-8f, 1.92596299112661746887e-8f)));
  float a, b;
  unpack2(y, a, b);
  asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(a));
  asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(b));
  return pack2(a, b);
}
// The largest of the elements of 16 bytes; NaN only if all are.
__device__ __forceinline__ float largest(const uint4& v, float) {
  return fmaxf(max3(__uint_as_float(v.x), __uint_as_float(v.y), __uint_as_float(v.z)), __uint_as_float(v.w));
}
__device__ __forceinline__ float largest(const uint4& v, __half) {
  auto h = [](const uint32_t& a) { return *reinterpret_cast<const __half2*>(&a); };
  const float2 f = __half22float2(__hmax2(__hmax2(h(v.x), h(v.y)), __hmax2(h(v.z), h(v.w))));
  return fmaxf(f.x, f.y);
}
__device__ __forceinline__ float largest(const uint4& v, __nv_bfloat16) {
  auto h = [](const uint32_t& a) { return *reinterpret_cast<const __nv_bfloat162*>(&a); };
  const float2 f = __bfloat1622float2(__hmax2(__hmax2(h(v.x), h(v.y)), __hmax2(h(v.z), h(v.w))));
  return fmaxf(f.x, f.y);
}

// The largest float below x (x finite or +infinity; -infinity stays).
__device__ __forceinline__ float float_below(float x) {
  if (x == 0.0f) return -__uint_as_float(1u);
  const unsigned int bits = __float_as_uint(x);
  if (bits == 0xFF800000u) return x;
  return __uint_as_float(bits >> 31 ? bits + 1 : bits - 1);
}

// The j-th largest of the lanes' values (j >= 1); equal ones count apart.
__device__ __forceinline__ float warp_jth(float x, int j) {
  const unsigned int bits = __float_as_uint(x + 0.0f);
  unsigned int up = bits >> 31 ? ~bits : bits | 0x80000000u, top = 0;
  for (; j > 0; --j) {
    top = __reduce_max_sync(0xFFFFFFFFu, up);
    const unsigned int who = __ballot_sync(0xFFFFFFFFu, up == top);
    if ((threadIdx.x & 31) == __ffs(who) - 1) up = 0;
  }
  return top == 0 ? -INFINITY : __uint_as_float(top >> 31 ? top & 0x7FFFFFFFu : ~top);
}

// A lower bound for the keep-th largest of the threads' values, where the first `warps` of the block have some: each has at
// least keep / warps at or above its own, and the smallest of these bounds is taken.  All threads call it.  Between this call and
// the next write to `scratch` lies a barrier: warps read it at the end.
__device__ __forceinline__ float block_bound(float x, int keep, int warps, float* scratch) {
  const float mine = warp_jth(x, (keep + warps - 1) / warps);
  if (threadIdx.x % 32 == 0) scratch[threadIdx.x / 32] = mine;
  __syncthreads();
  float bound = scratch[0];
#pragma unroll
  for (int w = 1; w < kBeamWarps; ++w) bound = w < warps ? fminf(bound, scratch[w]) : bound;
  return bound;
}

// Number of threads' counts, summed over the block.
__device__ __forceinline__ int block_sum(int c, int* counter) {
  c = __reduce_add_sync(0xFFFFFFFFu, c);
  if (threadIdx.x == 0) *counter = 0;
  __syncthreads();
  if (threadIdx.x % 32 == 0) atomicAdd(counter, c);
  __syncthreads();
  c = *counter;
  __syncthreads();
  return c;
}

// A tile with more candidates than a warp holds: the `keep` largest among the keys from before the tile (tokens below the
// tile's; segment w of `keys` has counts[w]) and the tile's logits, which are read once more.  They are dealt out to the
// segments in turn; returns the smallest.  The tile: vectors [base, end) of xv, the first logit of which is token `head`.
template <typename T>
__device__ __noinline__ unsigned long long thin_out_tile(unsigned long long* keys, const int* counts, int* counter, const uint4* xv, int base, int end,
                                                         int head, int keep) {
  constexpr int V = Vec16<T>::count, kScan = kBeamWarps * kBeamSegment / kBeamThreads;
  const int tid = threadIdx.x, first = head + base * V;
  unsigned long long before[kScan], least = 0;
#pragma unroll
  for (int i = 0; i < kScan; ++i) {
    const int at = i * kBeamThreads + tid;
    before[i] = at % kBeamSegment < counts[at / kBeamSegment] ? keys[at / kBeamSegment * kBeamStride + at % kBeamSegment] : 0;
    if (beam_key_token(before[i]) >= first) before[i] = 0;
  }
  // the logits are read anew in every pass: this is rare, and its registers would be the kernel's
  auto each = [&](auto&& f) {
#pragma unroll 1
    for (int u = 0; u < kBeamVectors; ++u) {
      const int at = base + u * kBeamThreads + tid;
      if (at >= end) break;
      float x[V];
      unpack16(xv[at], x, T());
#pragma unroll
      for (int e = 0; e < V; ++e) f(x[e] > -INFINITY ? beam_key(x[e], head + at * V + e) : 0ull);
    }
  };
  for (int bit = 63; bit >= 0; --bit) {
    const unsigned long long probe = least | 1ull << bit;
    int c = 0;
#pragma unroll
    for (int i = 0; i < kScan; ++i) c += before[i] >= probe;
    each([&](unsigned long long key) { c += key >= probe; });
    if (block_sum(c, counter) >= keep) least = probe;
  }
  if (tid == 0) *counter = 0;
  __syncthreads();
  auto add = [&](unsigned long long key) {
    if (key == 0 || key < least) return;
    const int at = atomicAdd(counter, 1);
    keys[at % kBeamWarps * kBeamStride + at / kBeamWarps] = key;
  };
#pragma unroll
  for (int i = 0; i < kScan; ++i) add(before[i]);
  each(add);
  __syncthreads();
  return least;
}

// More than kBeamRanked keys: leaves the `keep` largest at the front, in no order.
__device__ __noinline__ void thin_out(unsigned long long* keys, int n, int keep, int* counter) {
  constexpr int kMost = (kBeamCapacity + kBeamThreads - 1) / kBeamThreads;
  const int tid = threadIdx.x;
  unsigned long long mine[kMost], least = 0;
#pragma unroll
  for (int i = 0; i < kMost; ++i) mine[i] = i * kBeamThreads + tid < n ? keys[i * kBeamThreads + tid] : 0;
  for (int bit = 63; bit >= 0; --bit) {
    const unsigned long long probe = least | 1ull << bit;
    int c = 0;
#pragma unroll
    for (int i = 0; i < kMost; ++i) c += mine[i] >= probe;
    if (block_sum(c, counter) >= keep) least = probe;
  }
  if (tid == 0) *counter = 0;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kMost; ++i)
    if (mine[i] != 0 && mine[i] >= least) keys[atomicAdd(counter, 1)] = mine[i];
  __syncthreads();
}

// A block has part blockIdx.y of row blockIdx.x: `chunk` of its vectors, and with the first part the few logits in front of
// them, with the last those behind.
template <typename T, bool NORMALISE>
__global__ void __launch_bounds__(kBeamThreads, kBeamBlocks) beam_part_kernel(const BeamParams p) {
  extern __shared__ __align__(128) uint4 beam_tiles[];            // kBeamStages tiles
  __shared__ unsigned long long keys[kBeamCapacity];
  __shared__ uint64_t full[kBeamStages];
  __shared__ int counter, counts[kBeamWarps];
  __shared__ float bounds[kBeamWarps], maxima[kBeamWarps];     // the bound's are still read when a warp that is ahead has its row's maximum
  __shared__ double sums[kBeamWarps];
  __shared__ unsigned int abandoned;
  constexpr int V = Vec16<T>::count, U = kBeamVectors, kTile = kBeamThreads * U;
  constexpr uint32_t kNone = sizeof(T) == 4 ? 0xFF800000u : std::is_same<T, __half>::value ? 0xFC00FC00u : 0xFF80FF80u;     // -infinity
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  const int part = blockIdx.y, batch = static_cast<int>(blockIdx.x) / p.beams, beam = static_cast<int>(blockIdx.x) - batch * p.beams;
  if (tid == 0) {
    abandoned = 0;
    for (int s = 0; s < kBeamStages; ++s) mbar_init(&full[s], 1);
    fence_barrier_init();
    fence_proxy_async();
  }
  grid_dependency_wait();
  grid_dependency_launch();
  if (p.finished != nullptr && p.finished[batch * p.ld_finished + beam] != 0) return;

  const T* x = static_cast<const T*>(p.logits) + batch * p.batch_stride + beam * p.beam_stride;
  const int head = min(p.vocab, static_cast<int>(-(reinterpret_cast<uintptr_t>(x) / sizeof(T)) & (V - 1)));
  const int vectors = (p.vocab - head) / V, tail = p.vocab - head - vectors * V;
  const int v_begin = min(part * p.chunk, vectors), v_end = part == p.parts - 1 ? vectors : min(v_begin + p.chunk, vectors);
  const uint4* xv = reinterpret_cast<const uint4*>(x + head);
  auto copy = [&](int base, int stage) {                 // thread 0
    if (base >= v_end) return;
    const uint32_t bytes = static_cast<uint32_t>(min(kTile, v_end - base)) * 16;
    mbar_arrive_expect_tx(&full[stage], bytes);
    bulk_load(beam_tiles + stage * kTile, xv + base, bytes, &full[stage]);
  };
  if (tid == 0)
    for (int s = 0; s < kBeamStages; ++s) copy(v_begin + s * kTile, s);

  float m = -INFINITY, ref = -FLT_MAX;                   // this thread's maximum ...
  double sum = 0.0;                                      // ... and sum of exp(logit - ref)
  float above = -INFINITY, floor = -INFINITY;            // candidates are above `above`; of those found, `keep` reach `floor`
  int held = 0;                                          // candidates of this warp
  unsigned long long* segment = keys + warp * kBeamStride;
  __syncthreads();
  auto refer = [&] {
    if (m > ref + kBeamLag) {
      sum *= exp_of(ref - m);
      ref = m;
    }
  };
  // the few logits outside of whole vectors, one to a lane of the first warp: those in front first, those behind last, so
  // that of equal logits the ones met later always have the higher token
  auto take_one = [&](int at, bool mine) {
    const float value = mine ? to_float(x[at]) : -INFINITY;
    m = fmaxf(m, value);
    if constexpr (NORMALISE) {
      refer();
      sum += exp_of(value - ref);
    }
    const unsigned int who = __ballot_sync(0xFFFFFFFFu, value > above);
    if (value > above) segment[held + __popc(who & ((1u << lane) - 1))] = beam_key(value, at);      // there is room for them
    held += __popc(who);
  };
  if (part == 0 && head > 0 && warp == 0) take_one(lane, lane < head);
  int stage = 0, tile = 0;
  uint32_t parity = 0;
  for (int base = v_begin; base < v_end; base += kTile) {
    mbar_wait_or_abandon(&full[stage], parity, p.status, kDeviceTimeoutFull, &abandoned);
    uint4* here = beam_tiles + stage * kTile + tid;
    if (v_end - base < kTile)                            // the last tile: each thread fills up its own places
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (base + u * kBeamThreads + tid >= v_end) here[u * kBeamThreads] = make_uint4(kNone, kNone, kNone, kNone);
    float tops[U], top = -INFINITY;                      // not NaN
#pragma unroll
    for (int u = 0; u < U; ++u) {
      tops[u] = largest(here[u * kBeamThreads], T());
      top = fmaxf(top, tops[u]);
    }
    m = fmaxf(m, top);
    if constexpr (NORMALISE) {
      refer();
      const uint64_t minus = pack2(-ref, -ref);
      uint64_t s[2] = {0, 0};
#pragma unroll
      for (int u = 0; u < U; ++u) {
        float v[V];
        unpack16(here[u * kBeamThreads], v, T());
#pragma unroll
        for (int e = 0; e < V; e += 2) s[e / 2 % 2] = add2(s[e / 2 % 2], exp_of_pair(add2(pack2(v[e], v[e + 1]), minus)));
      }
      float a, b;
      unpack2(add2(s[0], s[1]), a, b);
      sum += a + b;
    }
    if ((tile & (tile - 1)) == 0) {
      const float bound = block_bound(m, p.keep, min((v_end - v_begin + 31) / 32, kBeamWarps), bounds);
      if (bound > floor) {
        floor = bound;
        above = float_below(bound);
      }
    }
    ++tile;
    if (__any_sync(0xFFFFFFFFu, top > above)) {
      // which of a lane's logits are candidates, then where its first goes: one scan for all of them (one for each logit, by a
      // ballot, took 2 us of the first tile)
      unsigned int in = 0;
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (__any_sync(0xFFFFFFFFu, tops[u] > above)) {
          float v[V];
          unpack16(here[u * kBeamThreads], v, T());
#pragma unroll
          for (int e = 0; e < V; ++e) in |= static_cast<unsigned int>(v[e] > above) << (u * V + e);
        }
      const int count = __popc(in);
      int at = count;
#pragma unroll
      for (int o = 1; o < 32; o *= 2) {
        const int before = __shfl_up_sync(0xFFFFFFFFu, at, o);
        if (lane >= o) at += before;
      }
      const int found = __shfl_sync(0xFFFFFFFFu, at, 31);
      for (at += held - count; in != 0; in &= in - 1, ++at) {
        const int which = __ffs(in) - 1, u = which / V, e = which % V;
        if (at < kBeamSegment)
          segment[at] = beam_key(to_float(reinterpret_cast<const T*>(here + u * kBeamThreads)[e]), head + (base + u * kBeamThreads + tid) * V + e);
      }
      held += found;
    }
    if (__syncthreads_or(held > kBeamSegment)) {
      // more than the warp holds (many equal logits, or ever larger ones): what follows lies further along the row, and equal
      // logits there lose
      if (lane == 0) counts[warp] = min(held, kBeamSegment);
      __syncthreads();
      floor = above = beam_key_logit(thin_out_tile<T>(keys, counts, &counter, xv, base, v_end, head, p.keep));
      held = (p.keep - warp + kBeamWarps - 1) / kBeamWarps;
    }
    // all have read the stage: the barrier above
    if (tid == 0) copy(base + kBeamStages * kTile, stage);
    if (++stage == kBeamStages) { stage = 0; parity ^= 1; }
  }
  if (part == p.parts - 1 && tail > 0 && warp == 0) take_one(p.vocab - tail + lane, lane < tail);

  // what reaches the floor, one after the other
  if (tile > 1) floor = fmaxf(floor, block_bound(m, p.keep, kBeamWarps, bounds));
  static_assert(kBeamCapacity * sizeof(unsigned long long) <= kBeamStages * kBeamTileBytes, "the tiles' place is used");
  unsigned long long* sorted = reinterpret_cast<unsigned long long*>(beam_tiles);
  constexpr int kMine = (kBeamStride + 31) / 32;
  unsigned long long mine[kMine];
  int left = 0, place[kMine];
  __syncwarp();
#pragma unroll
  for (int i = 0; i < kMine; ++i) {
    place[i] = -1;
    if (i * 32 >= held) continue;
    mine[i] = i * 32 + lane < held ? segment[i * 32 + lane] : 0;
    const bool in = mine[i] != 0 && beam_key_logit(mine[i]) >= floor;
    const unsigned int who = __ballot_sync(0xFFFFFFFFu, in);
    if (in) place[i] = left + __popc(who & ((1u << lane) - 1));
    left += __popc(who);
  }
  float all = m;
  if constexpr (NORMALISE) {
#pragma unroll
    for (int o = 16; o > 0; o /= 2) all = fmaxf(all, __shfl_xor_sync(0xFFFFFFFFu, all, o));
  }
  if (lane == 0) { counts[warp] = left; maxima[warp] = all; }
  __syncthreads();
  int n = 0, from = 0;
#pragma unroll
  for (int w = 0; w < kBeamWarps; ++w) {
    if (w == warp) from = n;
    n += counts[w];
    all = fmaxf(all, maxima[w]);
  }
#pragma unroll
  for (int i = 0; i < kMine; ++i)
    if (place[i] >= 0) sorted[from + place[i]] = mine[i];
  if constexpr (NORMALISE) {
    // a thread without a logit above -infinity has a sum of 0, or NaN
    double s = m == -INFINITY ? sum : sum * static_cast<double>(exp_of(ref - all));
#pragma unroll
    for (int o = 16; o > 0; o /= 2) s += __shfl_xor_sync(0xFFFFFFFFu, s, o);
    if (lane == 0) sums[warp] = s;
  }
  __syncthreads();
  const long long item = static_cast<long long>(blockIdx.x) * p.parts + part;
  if constexpr (NORMALISE) {
    if (tid == 0) {
      double s = sums[0];
      for (int w = 1; w < kBeamWarps; ++w) s += sums[w];
      p.part_max[item] = all;
      p.part_sum[item] = s;
    }
  }
  if (n > kBeamRanked) {
    thin_out(sorted, n, p.keep, &counter);
    n = p.keep;
  }
  unsigned long long* out = p.part_keys + item * p.keep;
  if (tid < n) {
    const unsigned long long key = sorted[tid];
    int rank = 0;
#pragma unroll 8
    for (int j = 0; j < n; ++j) rank += sorted[j] > key;
    if (rank < p.keep) out[rank] = key;
  } else if (tid < p.keep) {
    out[tid] = 0;
  }
}

// One block per search: log-sums of its prefixes, then the best of all parts' candidates.  A part's candidates are a sorted list
// of `keep`, and the values of all of them are worked out as whole numbers, beforehand.
//
// Up to 32 lists are merged by a warp, which takes the largest of their heads `keep` times: a chain of 0.1 us for each (one maximum
// over the warp).  With more lists that took two such chains, and the following is faster (5 searches of 91 lists, keep = 14: 11.9
// us for the step instead of 14.6; with 32 lists, keep = 8, 24.2 instead of 22.2): the lists' first entries, 64 or more, are
// compared with one another; the `keep`-th of these is a bound that `keep` candidates reach, and those of all lists that reach it
// are sorted by comparing all with all.  Where more than 256 reach it (most of them equal), and where the lists do not fit into
// shared memory, the warps share the lists.
//
// Whole numbers that order as the values do; 0 for -infinity and NaN.
__device__ __forceinline__ unsigned long long beam_order(double value) {
  if (!(value > -INFINITY)) return 0;
  const unsigned long long bits = __double_as_longlong(value + 0.0);
  return bits >> 63 ? ~bits : bits | 1ull << 63;
}
__device__ __forceinline__ double beam_ordered_value(unsigned long long order) {
  return __longlong_as_double(order >> 63 ? order & ~(1ull << 63) : ~order);
}
__device__ __forceinline__ unsigned long long warp_max(unsigned long long x) {
  const unsigned int hi = static_cast<unsigned int>(x >> 32), top = __reduce_max_sync(0xFFFFFFFFu, hi);
  const unsigned int low = __reduce_max_sync(0xFFFFFFFFu, hi == top ? static_cast<unsigned int>(x) : 0u);
  return static_cast<unsigned long long>(top) << 32 | low;
}
// A candidate of the merge; order is 0 behind the last of a list.
struct BeamEntry {
  unsigned long long order, key;
  int beam, pad;
};
// The lane whose entry comes first: by value, then the lower beam, then the larger key; -1 if no lane has one.
__device__ __forceinline__ int warp_first(const BeamEntry& e) {
  const unsigned int hi = static_cast<unsigned int>(e.order >> 32), top = __reduce_max_sync(0xFFFFFFFFu, hi);
  if (top == 0) return -1;                         // of a value above -infinity the upper half is not 0
  unsigned int who = __ballot_sync(0xFFFFFFFFu, hi == top);
  if (__popc(who) > 1) {
    const unsigned int lo = static_cast<unsigned int>(e.order), low = __reduce_max_sync(0xFFFFFFFFu, hi == top ? lo : 0u);
    bool in = hi == top && lo == low;
    who = __ballot_sync(0xFFFFFFFFu, in);
    if (__popc(who) > 1) {
      const int first = __reduce_min_sync(0xFFFFFFFFu, in ? e.beam : 0x7FFFFFFF);
      in = in && e.beam == first;
      const unsigned long long largest = warp_max(in ? e.key : 0ull);
      who = __ballot_sync(0xFFFFFFFFu, in && e.key == largest);
    }
  }
  return __ffs(who) - 1;
}

// A candidate in shared memory, without its key.
struct __align__(16) BeamMerged {
  unsigned long long order;
  int beam, pad;
};

// Takes `keep` times the lane's head that comes first; entry(at) is the lane's at-th (order 0 behind its last), and of equal ones of
// one beam key(at) decides.  taken[n] gets place(at), -1 behind the last.
template <typename Entry, typename Key, typename Place>
__device__ __forceinline__ void merge_heads(int* taken, int keep, Entry entry, Key key, Place place) {
  const int lane = threadIdx.x % 32;
  int at = 0, n = 0;
  BeamMerged e = entry(0), next = entry(1);
  for (; n < keep; ++n) {
    const unsigned int hi = static_cast<unsigned int>(e.order >> 32), top = __reduce_max_sync(0xFFFFFFFFu, hi);
    if (top == 0) break;                           // of a value above -infinity the upper half is not 0
    unsigned int who = __ballot_sync(0xFFFFFFFFu, hi == top);
    if ((who & (who - 1)) != 0) {
      const unsigned int lo = static_cast<unsigned int>(e.order), low = __reduce_max_sync(0xFFFFFFFFu, hi == top ? lo : 0u);
      bool in = hi == top && lo == low;
      who = __ballot_sync(0xFFFFFFFFu, in);
      if ((who & (who - 1)) != 0) {
        const int first = __reduce_min_sync(0xFFFFFFFFu, in ? e.beam : 0x7FFFFFFF);
        in = in && e.beam == first;
        const unsigned long long mine = in ? key(at) : 0ull, largest = warp_max(mine);
        who = __ballot_sync(0xFFFFFFFFu, in && mine == largest);
      }
    }
    if (lane == __ffs(who) - 1) {
      taken[n] = place(at);
      e = next;
      next = entry(++at + 1);
    }
  }
  for (n += lane; n < keep; n += 32) taken[n] = -1;
}

__host__ __device__ constexpr int beam_merge_scratch(int keep) {
  const int picked = kMergeThreads * static_cast<int>(sizeof(BeamMerged) + sizeof(unsigned long long));
  const int found = (1 + kMergeThreads / 32) * keep * static_cast<int>(sizeof(BeamEntry));
  return picked > found ? picked : found;
}

__global__ void __launch_bounds__(kMergeThreads) beam_merge_kernel(const BeamParams p) {
  extern __shared__ __align__(16) unsigned char beam_smem[];
  constexpr int kWarps = kMergeThreads / 32;
  const int lists = p.beams * p.parts, entries = lists * p.keep;                  // at most 1024 lists
  const bool merged = entries <= kBeamMergeMost && lists <= kMergeThreads;
  __shared__ unsigned int bound;
  __shared__ int n_picked;
  // A block is to fit beside the part kernel's blocks while it waits for them: what is not needed at a time lies in one place.
  BeamMerged* here = reinterpret_cast<BeamMerged*>(beam_smem);                    // [lists][keep], if they fit
  unsigned char* scratch = beam_smem + (merged ? entries * sizeof(BeamMerged) : 0);
  uint4* tops = reinterpret_cast<uint4*>(scratch);                                // first the entries that give the bound,
  BeamMerged* picked = reinterpret_cast<BeamMerged*>(scratch);                    // then those that reach it and their keys,
  unsigned long long* picked_key = reinterpret_cast<unsigned long long*>(picked + kMergeThreads);
  int* taken = reinterpret_cast<int*>(scratch);                                   // or [keep], as places in `here`,
  BeamEntry* found = reinterpret_cast<BeamEntry*>(scratch);                       // or [1 + warps][keep]: the result, what each warp found
  double* base = reinterpret_cast<double*>(scratch + beam_merge_scratch(p.keep)); // [beams]: score, less the log-sum
  unsigned char* place = reinterpret_cast<unsigned char*>(base + p.beams);        // [lists]: how far each has been taken
  unsigned char* done = place + lists;                                            // [beams]
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32, batch = blockIdx.x;
  grid_dependency_wait();
  grid_dependency_launch();
  const unsigned long long* far = p.part_keys + static_cast<long long>(batch) * entries;
  // the first of the keys come in while the log-sums are worked out
  constexpr int kMine = 4;
  unsigned long long keys[kMine];
#pragma unroll
  for (int i = 0; i < kMine; ++i) keys[i] = i * kMergeThreads + tid < entries ? far[i * kMergeThreads + tid] : 0;
  int group = 1;                   // lanes of a prefix, one for each of its parts (at most 32)
  while (group < p.parts) group *= 2;
  for (int b0 = warp * (32 / group); b0 < p.beams; b0 += kWarps * (32 / group)) {
    const int b = b0 + lane / group, i = lane % group;
    const bool mine = b < p.beams, some = mine && i < p.parts && p.normalise;    // an ended prefix has no sums: what is read for it is not used
    const long long item = (static_cast<long long>(batch) * p.beams + b) * p.parts + i;
    const float m = some ? p.part_max[item] : -INFINITY;
    double s = some ? p.part_sum[item] : 0.0, value = mine ? p.scores[batch * p.ld_scores + b] : 0.0;
    const bool ended = mine && p.finished != nullptr && p.finished[batch * p.ld_finished + b] != 0;
    if (p.normalise) {
      float all = m;
      for (int o = group / 2; o > 0; o /= 2) all = fmaxf(all, __shfl_xor_sync(0xFFFFFFFFu, all, o));
      if (m != all && m != -INFINITY) s *= exp(static_cast<double>(m) - static_cast<double>(all));
      for (int o = group / 2; o > 0; o /= 2) s += __shfl_xor_sync(0xFFFFFFFFu, s, o);
      if (!ended && i == 0) value -= (all == -INFINITY ? 0.0 : static_cast<double>(all)) + log(s);
    }
    if (mine && i == 0) { base[b] = value; done[b] = ended; }
  }
  __syncthreads();

  // entry `at` of list l of beam b; an ended prefix has one entry, in its first list
  auto work_out = [&](int l, int b, int at, unsigned long long key) {
    BeamEntry e = {0, key, b, 0};
    if (done[b]) {
      if (l == b * p.parts && at == 0) e = {beam_order(base[b]), static_cast<unsigned int>(~p.end_token), b, 0};
    } else if (key != 0) {
      e.order = beam_order(base[b] + static_cast<double>(beam_key_logit(key)));
    }
    return e;
  };
  auto put = [&](int n, unsigned long long order, int beam, int token) {
    const bool some = order != 0;
    p.out_scores[batch * p.ld_out_scores + n] = some ? static_cast<float>(beam_ordered_value(order)) : -INFINITY;
    p.parents[batch * p.ld_parents + n] = some ? beam : -1;
    p.tokens[batch * p.ld_tokens + n] = some ? token : -1;
  };
  if (merged) {
    auto enter = [&](int e, unsigned long long key) {
      const int l = e / p.keep, b = l / p.parts;
      here[e] = {work_out(l, b, e - l * p.keep, key).order, b, 0};
    };
#pragma unroll
    for (int i = 0; i < kMine; ++i)
      if (i * kMergeThreads + tid < entries) enter(i * kMergeThreads + tid, keys[i]);
    for (int e = kMine * kMergeThreads + tid; e < entries; e += kMergeThreads) enter(e, far[e]);
    if (tid == 0) {
      n_picked = 0;
      bound = 0xFFFFFFFFu;
    }
    __syncthreads();
    if (lists <= 32) {
      if (warp > 0) return;
      const int mine = lane * p.keep;
      const BeamMerged none = {0, -1, 0};
      merge_heads(taken, p.keep, [&](int at) { return lane < lists && at < p.keep ? here[mine + at] : none; }, [&](int at) { return far[mine + at]; },
                  [&](int at) { return mine + at; });
      __syncwarp();
      for (int i = lane; i < p.keep; i += 32) {
        const int from = taken[i];
        const BeamMerged e = from >= 0 ? here[from] : none;
        put(i, e.order, e.beam, from < 0 ? -1 : done[e.beam] ? p.end_token : beam_key_token(far[from]));
      }
      return;
    }
    const int depth = min(p.keep, max(1, max(64, 2 * p.keep) / lists)), items = lists * depth;
    const unsigned int top = tid < items ? static_cast<unsigned int>(here[tid / depth * p.keep + tid % depth].order >> 32) : 0;
    reinterpret_cast<unsigned int*>(tops)[tid] = top;
    __syncthreads();
    int above = 0;
#pragma unroll 4
    for (int j = 0; j < (items + 3) / 4; ++j) {
      const uint4 v = tops[j];
      above += (v.x > top) + (v.y > top) + (v.z > top) + (v.w > top);
    }
    const unsigned int least = __reduce_min_sync(0xFFFFFFFFu, tid < items && above < p.keep ? top : 0xFFFFFFFFu);
    if (lane == 0) atomicMin(&bound, least);
    __syncthreads();
    const unsigned int reached = max(bound, 1u);   // of a value above -infinity the upper half is not 0
    auto pick = [&](int e, auto&& key) {           // one entry of each thread, or none
      const bool in = e < entries && static_cast<unsigned int>(here[e].order >> 32) >= reached;
      const unsigned int who = __ballot_sync(0xFFFFFFFFu, in);
      if (who == 0) return;
      int at = 0;
      if (lane == 0) at = atomicAdd(&n_picked, __popc(who));
      at = __shfl_sync(0xFFFFFFFFu, at, 0) + __popc(who & ((1u << lane) - 1));
      if (in && at < kMergeThreads) {
        picked[at] = here[e];
        picked_key[at] = key();
      }
    };
#pragma unroll
    for (int i = 0; i < kMine; ++i)
      if (i * kMergeThreads < entries) pick(i * kMergeThreads + tid, [&] { return keys[i]; });
    for (int e = kMine * kMergeThreads + tid; e - tid < entries; e += kMergeThreads) pick(e, [&] { return far[e]; });
    __syncthreads();
    const int n = n_picked;
    if (n <= kMergeThreads) {
      int share = 1;               // threads of a candidate, each of which compares it with some of the others
      while (share < 32 && 2 * share * n <= kMergeThreads) share *= 2;
      const int i = min(tid / share, n - 1);
      if (n > 0) {
        const BeamMerged mine = picked[i];
        const unsigned long long key = picked_key[i];
        int rank = 0;
#pragma unroll 4
        for (int j = tid % share; j < n; j += share) {
          const BeamMerged other = picked[j];
          const bool first = (other.beam < mine.beam) | ((other.beam == mine.beam) & (picked_key[j] > key));
          rank += (other.order > mine.order) | ((other.order == mine.order) & first);
        }
        for (int o = share / 2; o > 0; o /= 2) rank += __shfl_xor_sync(0xFFFFFFFFu, rank, o);
        if (tid < n * share && tid % share == 0 && rank < p.keep) put(rank, mine.order, mine.beam, done[mine.beam] ? p.end_token : beam_key_token(key));
      }
      for (int left = n + tid; left < p.keep; left += kMergeThreads) put(left, 0, -1, -1);
      return;
    }
  }

  // The warps share the lists, a warp takes the largest head of its own `keep` times, and the first merges what they found.
  auto entry_of = [&](int l, int b, int at) {
    return at < p.keep ? work_out(l, b, at, far[static_cast<long long>(l) * p.keep + at]) : BeamEntry{0, 0, b, 0};
  };
  const BeamEntry none = {0, 0, -1, 0};
  BeamEntry* result = found;
  found += p.keep;
  const int first = static_cast<int>(static_cast<long long>(lists) * warp / kWarps), last = static_cast<int>(static_cast<long long>(lists) * (warp + 1) / kWarps);
  for (int l = first + lane; l < last; l += 32) place[l] = 0;
  BeamEntry best;
  int from;
  auto look = [&] {                // the lane's first entry
    best = none;
    from = -1;
    for (int l = first + lane; l < last; l += 32) {
      const BeamEntry e = entry_of(l, l / p.parts, place[l]);
      if (e.order > best.order || (e.order != 0 && e.order == best.order && e.beam == best.beam && e.key > best.key)) { best = e; from = l; }
    }
  };
  look();
  int n = 0;
  for (; n < p.keep; ++n) {
    const int who = warp_first(best);
    if (who < 0) break;
    if (lane == who) {
      found[warp * p.keep + n] = best;
      ++place[from];
      look();
    }
  }
  for (n += lane; n < p.keep; n += 32) found[warp * p.keep + n] = none;
  __syncthreads();
  if (warp > 0) return;
  int at = 0;                      // lane w: how far list w of `found` has been taken
  BeamEntry e = lane < kWarps ? found[lane * p.keep] : none;
  for (int i = 0; i < p.keep; ++i) {
    const int who = warp_first(e);
    if (who < 0 ? lane == 0 : lane == who) result[i] = e;
    if (lane == who) e = ++at < p.keep ? found[lane * p.keep + at] : none;
  }
  __syncwarp();
  for (int i = lane; i < p.keep; i += 32) put(i, result[i].order, result[i].beam, beam_key_token(result[i].key));
}

}  // namespace cuasr_b200
