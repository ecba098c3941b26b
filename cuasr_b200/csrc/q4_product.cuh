// Plus-times product of a few rows with weights in 4 bits: Y = X W^T, W = scale (q - zero) by groups along k.
//
// The weights are read once, so the floor is their bytes at the memory's rate; at 6.5 TB/s that is 46 weights per SM and
// clock, which leaves about ten instructions of a lane for eight weights.  Hence the tensor cores do the products
// (mma.sync m16n8k16: sixteen weight rows by up to eight rows of X; an eighth of a tile is enough for one row, and the
// instruction is not what bounds the kernel), and two weights become factors by an AND and one multiply-add.  As the last bits of a
// 16-bit number four bits are the subnormal q u, four places further up 16 q u, both exact (u = 2^-24 in binary16; 2^-133 in bfloat16,
// where the numbers up to 255 u, the first normal ones among them, are still evenly spaced); times a power of two and less the zero
// point they are (q - z) e, an exact number as well (e = 2^-9, 2^-6).  So the sums are those of the formula, in units of e: a
// weight at its zero point adds nothing, and infinities and NaN of X go where the formula has them.  (Leaving zero points out of the products,
// sum x q - z sum x, would save the multiply-add, but round against sum |x| q instead of sum |x (q - z)|.)
//
// A 32-bit X is staged as three columns of 8 bits each, which sum up to it exactly (bits below 2^-133 are lost).
//
// The order of k inside a product is free as long as both operands have it.  A 32-bit word holds k, k + 1, ... k + 7; its
// AND-OR yields the pairs (k, k + 4), (k + 1, k + 5), ...  So a lane takes whole words of a weight row as they lie, and X is
// laid out in shared memory, once per block, in the order that matches.
//
// A worker of 1, 2, 4 or 8 warps has 32 weight rows at a time, or 16 where X has more than eight columns (whose sums take the
// registers: 32 rows by 32 columns leave room for eight warps of an SM, 16 rows for sixteen; 4096 x 4096 by 32 rows of X 14.2 us
// instead of 16.1).  Its warps take the steps of 256 k in turn and put their sums together in shared memory.  Workers do not wait for
// one another (but for clusters, below).  Every warp has a pipeline of its own: its steps (4 KB, or 2) come into its two stages by
// TMA, issued by its first lane as soon as a stage has been read, across the ends of a worker's rows too, so that the memory does not
// wait for sums.  Weight rows that TMA cannot describe (not on 16-byte boundaries) are copied by the lanes in aligned words (cp.async)
// and shifted into place when they are read.
//
// Where there are few weight rows for the SMs, or X is too large for a block's shared memory, the blocks of a cluster share k, and
// their sums meet through distributed shared memory.
//
// What bounds it: for large n the instructions of a step (eight rows, 128000 x 4096, weights that are not in L2: 65 us, 4.2 TB/s; the
// issue slots are 57 % full, the pipe that does the ANDs 49 %); with more columns of X the chain of a warp's instructions (32 rows, 8192 x 8192:
// 32.6 us), neither their number, nor the products (a third of the
// rate of mma.sync), nor the reads of X, each of which was taken out in a trial without a gain; for small n what precedes the products
// (the launch, X laid out: 2 to 8 us).  Pairs of times in this file compare two choices as the kernel was when one was made; times change by
// 5 % either way with what has been mended since.  Tried and slower: three stages, one box of 128 bytes instead of two of 64, clusters of eight
// (15 run at a time: 32 rows, 8192 x 8192 57 us instead of 35), more loads of X in flight (the registers: 57 us
// with four of a warp instead of two), all products of one pair before those of the other (63 instead of 61).
#pragma once

#include "../../include/cuasr_b200_types.h"
#include "decode_types.cuh"

namespace cuasr_b200 {

constexpr int kQ4Step = 256;                  // k of a step, two halves of 16 words of a weight row, 4 of them to a lane
constexpr int kQ4Pitch = kQ4Step / 2 + 4;     // bytes between rows of a stage that the lanes fill: one more aligned word
// Weight rows of a worker are RT tiles of the instruction.
template <bool TMA, int RT> constexpr int kQ4Stage = 16 * RT * (TMA ? kQ4Step / 2 : kQ4Pitch);
constexpr int kQ4Stages = 2;                  // of a warp; three measured slower (128000 x 4096 read alone: 53 us instead of 45)
constexpr int kQ4SliceChoices = 3;            // 1, 2 or 4 blocks of a cluster share k
constexpr int kQ4SumPad = 4;                  // floats between columns of a warp's sums, besides its rows: no bank twice

struct Q4Params {
  const void* X; long long ldx;
  const unsigned char* W; long long ldw;
  const void* scales; long long ld_scales;
  const unsigned char* zeros; long long ld_zeros;
  void* Y; long long ldy;
  int m, n, k, group, groups, group_shift;    // group_shift: log2(group), or -1
  int type_x, type_y, type_scale;             // cuasr_dtype_t
  int rows;                                   // rows of X of a pass (blockIdx.y)
  int units, parts, slices;                   // 16 RT weight rows each; warps of a worker; blocks that share k
  int panel_steps;                            // steps whose X fits into shared memory; a multiple of parts if not all
  int sum_bytes;
  unsigned int* status;
  bool x_vectors;                             // X can be read 16 bytes at a time
};

__device__ __forceinline__ void store_real(void* base, long long at, int type, float v) {
  if (type == CUASR_F32) static_cast<float*>(base)[at] = v;
  else if (type == CUASR_F16) static_cast<__half*>(base)[at] = __float2half_rn(v);
  else static_cast<__nv_bfloat16*>(base)[at] = __float2bfloat16_rn(v);
}

// d = c + a b of a 16 x 16 and a 16 x 8 tile.
template <bool BF16>
__device__ __forceinline__ void mma_16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, float c0, float c1, float c2, float c3) {
  if constexpr (BF16)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c0), "f"(c1), "f"(c2), "f"(c3));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c0), "f"(c1), "f"(c2), "f"(c3));
}

// e: what q - z is multiplied by in a factor.
template <bool BF16> constexpr float kQ4Unit = BF16 ? 0.015625f : 0.001953125f;       // 2^-6, 2^-9

// a b + c of pairs; subnormal numbers are kept.
template <bool BF16>
__device__ __forceinline__ uint32_t fma_pair(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t r;
  if constexpr (BF16) asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
  else asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
  return r;
}
// The pair (v, v) of a whole number of units, at most 15 either way.
template <bool BF16>
__device__ __forceinline__ uint32_t unit_pair(int v) {
  const float x = static_cast<float>(v) * kQ4Unit<BF16>;
  if constexpr (BF16) return (__float_as_uint(x) >> 16) * 0x10001u;
  else return __half_as_ushort(__float2half_rn(x)) * 0x10001u;
}
// The factors of the pairs (k, k + 4) ... (k + 3, k + 7) of a word; minus_z: unit_pair(-z).
template <bool BF16>
__device__ __forceinline__ void factors_of(uint32_t w, uint32_t minus_z, uint32_t (&out)[4]) {
  constexpr uint32_t kUp = BF16 ? 0x7F007F00u : 0x78007800u, kUp16 = BF16 ? 0x7D007D00u : 0x68006800u;      // e / u, e / (16 u)
  const uint32_t upper = w >> 8;
  out[0] = fma_pair<BF16>(w & 0x000F000Fu, kUp, minus_z);
  out[1] = fma_pair<BF16>(w & 0x00F000F0u, kUp16, minus_z);
  out[2] = fma_pair<BF16>(upper & 0x000F000Fu, kUp, minus_z);
  out[3] = fma_pair<BF16>(upper & 0x00F000F0u, kUp16, minus_z);
}

// Memory word of half a step that word i of lane t of a quad is.  A group's products are summed apart, so the four lanes of an
// instruction share a group: LW words in a row go to a lane, 4 where groups are whole steps, 2 for groups of 64, 1 for 32.
template <int LW>
__device__ __forceinline__ int word_index(int i, int t) {
  return LW == 4 ? t * 4 + i : LW == 2 ? (i / 2) * 8 + t * 2 + i % 2 : i * 4 + t;
}

// Half a stage holds its rows 64 bytes apart, their four 16-byte chunks exchanged as TMA's 64-byte swizzle does it: the
// words that eight rows and four lanes read at a time lie in different banks.
__device__ __forceinline__ int chunk_at(int row, int chunk) { return row * 64 + ((chunk ^ (row >> 1 & 3)) << 4); }

// Words 0 .. 3 of lane (g, t) from row g + 8 j of half a stage.
template <int LW>
__device__ __forceinline__ void read_words(uint32_t (&w)[4], const unsigned char* half, int j, int g, int t) {
  const unsigned char* row = half + j * 512;
  if constexpr (LW == 4) {
    const uint4 v = *reinterpret_cast<const uint4*>(row + chunk_at(g, t));
    w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
  } else if constexpr (LW == 2) {
#pragma unroll
    for (int i = 0; i < 4; i += 2) {
      const uint2 v = *reinterpret_cast<const uint2*>(row + chunk_at(g, i + t / 2) + t % 2 * 8);
      w[i] = v.x; w[i + 1] = v.y;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = *reinterpret_cast<const uint32_t*>(row + chunk_at(g, i) + t * 4);
  }
}
// ... from a stage that the lanes filled, whose row j starts `shift` / 8 bytes into its first word.
template <int LW>
__device__ __forceinline__ void read_words_shifted(uint32_t (&w)[4], const unsigned char* half, int j, int g, int t, unsigned int shift) {
  const uint32_t* row = reinterpret_cast<const uint32_t*>(half + (j * 8 + g) * kQ4Pitch);
#pragma unroll
  for (int i = 0; i < 4; i += LW) {
    const int first = word_index<LW>(i, t);
    uint32_t v = row[first];
#pragma unroll
    for (int e = 0; e < LW; ++e) {
      const uint32_t more = row[first + e + 1];
      w[i + e] = __funnelshift_r(v, more, shift);
      v = more;
    }
  }
}

// The lanes' way to copy a step: lane l has word l of every row, lane r also the last word (of 33) of row r.  Words reach over the
// ends of a row into its neighbours'; those that would reach outside of [W, last) are put together from its bytes.
__device__ __forceinline__ void copy_word(const Q4Params& p, unsigned char* stage, long long row, int step, int r, int word, int row_bytes,
                                          const unsigned char* last) {
  unsigned char* to = stage + r * kQ4Pitch + word * 4;
  const unsigned char* q = p.W + row * p.ldw + static_cast<long long>(step) * (kQ4Step / 2);
  const int off = static_cast<int>(reinterpret_cast<uintptr_t>(q) & 3);
  const int at = step * (kQ4Step / 2) + word * 4 - off;         // of the row
  if (row >= p.n || at >= row_bytes) {
    *reinterpret_cast<uint32_t*>(to) = 0;
    return;
  }
  const unsigned char* a = q - off + word * 4;
  if (a >= p.W && a + 4 <= last) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(to)), "l"(a) : "memory");
  } else {
    uint32_t v = 0;
    for (int b = 0; b < 4; ++b)
      if (a + b >= p.W && a + b < last) v |= static_cast<uint32_t>(a[b]) << (8 * b);
    *reinterpret_cast<uint32_t*>(to) = v;
  }
}
template <int RT>
__device__ __forceinline__ void copy_step(const Q4Params& p, unsigned char* stage, long long first_row, int step, int lane, int row_bytes,
                                          const unsigned char* last) {
  const unsigned char* q = p.W + first_row * p.ldw + static_cast<long long>(step) * (kQ4Step / 2);
  constexpr int kRows = 16 * RT;
  if (first_row + kRows <= p.n && q - 3 >= p.W && q + (kRows - 1) * p.ldw + kQ4Step / 2 + 4 <= last) {
    // every word lies inside the operand; what lies behind a row's end meets zeros of X
    const uint32_t to = smem_u32(stage) + lane * 4;
#pragma unroll 8
    for (int r = 0; r < kRows; ++r) {
      const unsigned char* a = q - (reinterpret_cast<uintptr_t>(q) & 3) + lane * 4;
      asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(to + r * kQ4Pitch), "l"(a) : "memory");
      q += p.ldw;
    }
    if (lane >= kRows) return;
    const unsigned char* mine = p.W + (first_row + lane) * p.ldw + static_cast<long long>(step) * (kQ4Step / 2);
    const unsigned char* a = mine - (reinterpret_cast<uintptr_t>(mine) & 3) + 128;
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(stage) + lane * kQ4Pitch + 128), "l"(a) : "memory");
    return;
  }
#pragma unroll 1
  for (int r = 0; r < kRows; ++r) copy_word(p, stage, first_row + r, step, r, lane, row_bytes, last);
  if (lane < kRows) copy_word(p, stage, first_row + lane, step, lane, 32, row_bytes, last);
}

// Eight values of a row of X from k on, zeros from p.k on: E = uint32_t for 32-bit rows, unsigned short for 16-bit ones.
template <typename E>
__device__ __forceinline__ void load_x8(const Q4Params& p, long long row, int k, uint32_t (&x)[2 * sizeof(E)]) {
  const E* at = static_cast<const E*>(p.X) + row * p.ldx + k;
  if (p.x_vectors && k + 8 <= p.k) {
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(E)) / 2; ++i) {
      const uint4 v = reinterpret_cast<const uint4*>(at)[i];
      x[4 * i] = v.x; x[4 * i + 1] = v.y; x[4 * i + 2] = v.z; x[4 * i + 3] = v.w;
    }
  } else {
    uint32_t e[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) e[i] = k + i < p.k ? at[i] : 0u;
#pragma unroll
    for (int i = 0; i < 2 * static_cast<int>(sizeof(E)); ++i) x[i] = sizeof(E) == 4 ? e[i] : e[2 * i % 8] | e[(2 * i + 1) % 8] << 16;
  }
}

// Lays out X for steps [begin, end): 16 bytes for each (half a step, word of a lane, column, lane of a quad).  Columns are the rows of
// X; a 32-bit row is three.
// Not inlined: it runs once a panel, and its registers are not to crowd out those of the products.
template <typename E, int LW, int THREADS>
__device__ __noinline__ void stage_x(const Q4Params& p, uint4* xs, int r0, int rows, int columns, int begin, int end) {
  constexpr int kBatch = 4 / sizeof(E);                       // loads of as many items are in flight: more cost the kernel registers
  constexpr int kAtOnce = THREADS / 32;
  const int lane = threadIdx.x % 32, steps = end - begin, in_half = lane % 16;
  const int i = LW == 4 ? in_half % 4 : LW == 2 ? in_half / 8 * 2 + in_half % 2 : in_half / 4;
  const int t = LW == 4 ? in_half / 4 : LW == 2 ? in_half / 2 % 4 : in_half % 4;
  uint4* const xs_lane = xs + (lane / 16 * 4 + i) * columns * 4 + t;
  // a warp takes a step of a row (32 words) at a time: row r, step s behind `begin`
  int r = threadIdx.x / 32 / steps, s = threadIdx.x / 32 % steps;
  auto next = [&](int& row, int& step) {
    step += kAtOnce;
    while (step >= steps) { step -= steps; ++row; }
  };
  while (r < rows) {
    uint32_t bits[kBatch][2 * sizeof(E)];
    int row = r, step = s;
#pragma unroll
    for (int q = 0; q < kBatch; ++q) {
      if (row < rows) load_x8<E>(p, r0 + row, (begin + step) * kQ4Step + lane * 8, bits[q]);
      next(row, step);
    }
#pragma unroll
    for (int q = 0; q < kBatch; ++q) {
      if (r >= rows) break;
      uint4* to = xs_lane + (s * 8 * columns + r) * 4;
      if constexpr (sizeof(E) == 2) {
        const uint32_t(&v)[4] = bits[q];
        *to = make_uint4(__byte_perm(v[0], v[2], 0x5410), __byte_perm(v[0], v[2], 0x7632), __byte_perm(v[1], v[3], 0x5410),
                         __byte_perm(v[1], v[3], 0x7632));
      } else {
        uint32_t h[3][8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          // the upper half is a bfloat16, rounded towards zero; what is left of an infinity or a NaN is nothing (a NaN stays one
          // whichever of its bits are set)
          const uint32_t all = bits[q][e];
          const bool finite = (all & 0x7F800000u) != 0x7F800000u;
          h[0][e] = finite || (all & 0x007FFFFFu) == 0 ? all >> 16 : 0x7FFFu;
          float rest = finite ? __uint_as_float(all) - __uint_as_float(all & 0xFFFF0000u) : 0.0f;
          h[1][e] = __float_as_uint(rest) >> 16;
          rest -= __uint_as_float(h[1][e] << 16);
          h[2][e] = __float_as_uint(rest) >> 16;
        }
#pragma unroll
        for (int part = 0; part < 3; ++part)
          to[part * rows * 4] = make_uint4(h[part][0] | h[part][4] << 16, h[part][1] | h[part][5] << 16, h[part][2] | h[part][6] << 16,
                                           h[part][3] | h[part][7] << 16);
      }
      next(r, s);
    }
  }
}

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_barrier() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ float load_cluster(const float* mine, uint32_t rank) {
  uint32_t at;
  float v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_u32(mine)), "r"(rank));
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory");
  return v;
}

__device__ __forceinline__ void worker_barrier(int worker, int warps) {
  asm volatile("bar.sync %0, %1;" ::"r"(worker + 1), "r"(warps * 32) : "memory");
}

// NT tiles of eight columns of X.  WARPS: 16, or 8 where the sums of more than eight columns take the registers or X the shared
// memory.
template <bool BF16, int NT, int RT, int WARPS, int LW, bool TMA, bool ZEROS>
__global__ void __launch_bounds__(32 * WARPS, 1)
q4_kernel(const __grid_constant__ CUtensorMap map, const __grid_constant__ Q4Params p) {
  extern __shared__ __align__(1024) unsigned char q4_smem[];
  constexpr int kThreads = 32 * WARPS, kRows = 16 * RT, kStage = kQ4Stage<TMA, RT>, kSumStride = kRows + kQ4SumPad, kBuffer = NT * 8 * kSumStride;
  __shared__ uint64_t full[WARPS][kQ4Stages];
  __shared__ unsigned int abandoned;
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32, g = lane / 4, t = lane % 4;
  const int parts = p.parts, part_of = warp % parts, local = warp / parts, workers_here = WARPS / parts;
  unsigned char* stages = q4_smem + warp * kQ4Stages * kStage;
  float* all_sums = reinterpret_cast<float*>(q4_smem + WARPS * kQ4Stages * kStage);
  const int buffers = max(parts - 1, 1);                   // of a worker
  float* sums = all_sums + local * buffers * kBuffer;
  uint4* xs = reinterpret_cast<uint4*>(reinterpret_cast<unsigned char*>(all_sums) + p.sum_bytes);
  const int slice = p.slices > 1 ? static_cast<int>(cluster_rank()) : 0;
  const int r0 = blockIdx.y * p.rows, rows = min(p.rows, p.m - r0);
  const int columns = p.type_x == CUASR_F32 ? 3 * rows : rows;
  const int all_steps = (p.k + kQ4Step - 1) / kQ4Step;
  const int begin = static_cast<int>(static_cast<long long>(all_steps) * slice / p.slices);
  const int end = static_cast<int>(static_cast<long long>(all_steps) * (slice + 1) / p.slices);
  const bool one_panel = end - begin <= p.panel_steps;
  // In more than one round neighbouring units are in different blocks, so that the last, which need not be full, leaves every SM as
  // much to do (eight rows, 128000 x 4096 in a graph: 57 us instead of 60.7); in one round in the same block (32 rows, 8192 x 8192: 34.9 us
  // instead of 36.3).
  const int clusters = static_cast<int>(gridDim.x) / p.slices, cluster = static_cast<int>(blockIdx.x) / p.slices;
  const int workers = clusters * workers_here, rounds = (p.units + workers - 1) / workers;
  auto worker_of = [&](int l) { return rounds > 1 ? l * clusters + cluster : cluster * workers_here + l; };
  const int worker = worker_of(local);

  if constexpr (TMA) {
    if (lane == 0) {
      for (int s = 0; s < kQ4Stages; ++s) mbar_init(&full[warp][s], 1);
      fence_barrier_init();
      fence_proxy_async();
    }
  }
  if (tid == 0) abandoned = 0;
  __syncthreads();
  grid_dependency_wait();
  grid_dependency_launch();

  // what comes next into the pipeline: step `ahead` of unit `ahead_unit`, into stage `ahead_stage`
  int ahead_unit = begin + part_of < end ? worker : p.units, ahead = begin + part_of, ahead_stage = 0;
  const int row_bytes = (p.k + 1) / 2;
  auto copy_ahead = [&] {           // TMA: lane 0 alone
    if (ahead_unit < p.units) {
      unsigned char* to = stages + ahead_stage * kStage;
      if constexpr (TMA) {
        uint64_t* bar = &full[warp][ahead_stage];
        const int y = ahead_unit * kRows, x = ahead * (kQ4Step / 2);
        mbar_arrive_expect_tx(bar, kStage);
        tma_load_2d(to, &map, bar, x, y);
        tma_load_2d(to + kStage / 2, &map, bar, x + kQ4Step / 4, y);
      } else {
        copy_step<RT>(p, to, static_cast<long long>(ahead_unit) * kRows, ahead, lane, row_bytes, p.W + (p.n - 1) * p.ldw + row_bytes);
      }
      ahead += parts;
      if (ahead >= end) { ahead = begin + part_of; ahead_unit += workers; }
      if (++ahead_stage == kQ4Stages) ahead_stage = 0;
    }
    if constexpr (!TMA) asm volatile("cp.async.commit_group;" ::: "memory");
  };
  if (!TMA || lane == 0)
    for (int s = 0; s < kQ4Stages; ++s) copy_ahead();

  // Scales and zero points of a step, loaded one step ahead, for both its halves.  Where half a step has one group, lane
  // (g, t) has those of row t * 8 + g (of two tiles; of one, t and t + 2 have the same); else those of its t-th group for rows g, 8 + g, ...
  constexpr int kMine = LW == 4 ? 1 : 2 * RT;
  uint32_t next_scale[2][kMine], next_zero[2][kMine];
  const int scale_shift = p.type_scale == CUASR_BF16 ? 16 : 0;
  auto load_scales = [&](int unit, int step) {
    if (unit >= p.units || step >= end) return;
    // the bits are converted where they are used, so that nothing waits here
    int group[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int k = step * kQ4Step + u * (kQ4Step / 2) + (LW == 4 ? 0 : LW == 2 ? t / 2 * 64 : t * 32);
      group[u] = min(p.group_shift >= 0 ? k >> p.group_shift : k / p.group, p.groups - 1);
    }
#pragma unroll
    for (int j = 0; j < kMine; ++j) {
      const long long row = min(unit * kRows + (LW == 4 ? t % (2 * RT) : j) * 8 + g, p.n - 1);      // rows behind the last get the last one's
      const long long at = row * p.ld_scales;
      if (p.type_scale == CUASR_F32) {
#pragma unroll
        for (int u = 0; u < 2; ++u) next_scale[u][j] = __ldg(static_cast<const unsigned int*>(p.scales) + at + group[u]);
      } else {
#pragma unroll
        for (int u = 0; u < 2; ++u) next_scale[u][j] = __ldg(static_cast<const unsigned short*>(p.scales) + at + group[u]);
      }
      if constexpr (ZEROS) {
#pragma unroll
        for (int u = 0; u < 2; ++u) next_zero[u][j] = __ldg(p.zeros + row * p.ld_zeros + group[u]);
      }
    }
  };
  load_scales(worker, begin + part_of);

  int stage = 0;
  uint32_t parity = 0;
  for (int round = 0; round < rounds; ++round) {
    const int unit = worker + round * workers;
    const bool mine = unit < p.units;
    // rows that do not start on a word: how far into it, the same for every step
    unsigned int shift[TMA ? 1 : 2 * RT];
    if constexpr (!TMA) {
#pragma unroll
      for (int j = 0; j < 2 * RT; ++j)
        shift[j] = static_cast<unsigned int>((reinterpret_cast<uintptr_t>(p.W) + (static_cast<long long>(unit) * kRows + j * 8 + g) * p.ldw) & 3) * 8;
    }
    float acc[RT][NT][4] = {};
    for (int panel = begin; panel < end; panel += p.panel_steps) {
      const int panel_end = min(end, panel + p.panel_steps);
      if (!one_panel || round == 0) {
        if (!one_panel) __syncthreads();       // the panel before has been read
        if (BF16 && p.type_x == CUASR_F32) stage_x<uint32_t, LW, kThreads>(p, xs, r0, rows, columns, panel, panel_end);
        else stage_x<unsigned short, LW, kThreads>(p, xs, r0, rows, columns, panel, panel_end);
        __syncthreads();
      }
      if (!mine) continue;
      for (int step = panel + part_of; step < panel_end; step += parts) {
        float scale[2][kMine];
        uint32_t zero[2][kMine];
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int j = 0; j < kMine; ++j) {
            scale[u][j] = p.type_scale == CUASR_F16 ? __half2float(__ushort_as_half(static_cast<unsigned short>(next_scale[u][j])))
                                                    : __uint_as_float(next_scale[u][j] << scale_shift);
            if constexpr (ZEROS) zero[u][j] = unit_pair<BF16>(-static_cast<int>(next_zero[u][j] & 15u));
          }
        if (step + parts < end) load_scales(unit, step + parts);
        else load_scales(unit + workers, begin + part_of);
        if constexpr (TMA) {
          mbar_wait_or_abandon(&full[warp][stage], parity, p.status, kDeviceTimeoutFull, &abandoned);
        } else {
          asm volatile("cp.async.wait_group %0;" ::"n"(kQ4Stages - 1) : "memory");
          __syncwarp();
        }
#pragma unroll (NT == 4 ? 1 : 2)             // of 32 columns both halves' words do not fit into the registers
        for (int u = 0; u < 2; ++u) {
          const unsigned char* words = stages + stage * kStage + (TMA ? u * kStage / 2 : u * kQ4Step / 4);
          const uint4* x = xs + (((step - panel) * 2 + u) * 16 * columns + lane);
          uint32_t w[2 * RT][4];
#pragma unroll
          for (int j = 0; j < 2 * RT; ++j) {
            if constexpr (TMA) read_words<LW>(w[j], words, j, g, t);
            else read_words_shifted<LW>(w[j], words, j, g, t, shift[j]);
          }
          float part[RT][NT][4], f[2 * RT];
          uint32_t minus_z[2 * RT];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            if (i % LW == 0) {
#pragma unroll
              for (int j = 0; j < 2 * RT; ++j) {
                const int from = (lane & ~3) + (LW == 4 ? j : LW == 2 ? i / 2 * 2 : i), of = LW == 4 ? 0 : j;
                f[j] = __shfl_sync(0xFFFFFFFFu, scale[u][of], from);
                if constexpr (ZEROS) minus_z[j] = __shfl_sync(0xFFFFFFFFu, zero[u][of], from);
                else minus_z[j] = BF16 ? 0xBE00BE00u : 0xA400A400u;            // -8 e
              }
            }
            uint4 b[NT];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
              b[nt] = x[(i * columns + nt * 8) * 4];        // behind the last column: whatever follows, in columns nobody reads
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
              uint32_t lo[4], hi[4];
              factors_of<BF16>(w[2 * rt][i], minus_z[2 * rt], lo);
              factors_of<BF16>(w[2 * rt + 1][i], minus_z[2 * rt + 1], hi);
              const uint32_t a0[4] = {lo[0], hi[0], lo[1], hi[1]}, a1[4] = {lo[2], hi[2], lo[3], hi[3]};
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) {
                float(&d)[4] = part[rt][nt];
                if (i % LW == 0) mma_16816<BF16>(d, a0, b[nt].x, b[nt].y, 0.0f, 0.0f, 0.0f, 0.0f);
                else mma_16816<BF16>(d, a0, b[nt].x, b[nt].y, d[0], d[1], d[2], d[3]);
                mma_16816<BF16>(d, a1, b[nt].z, b[nt].w, d[0], d[1], d[2], d[3]);
                if (i % LW == LW - 1) {
#pragma unroll
                  for (int c = 0; c < 4; ++c) acc[rt][nt][c] = fmaf(f[2 * rt + c / 2], d[c], acc[rt][nt][c]);
                }
              }
            }
          }
        }
        __syncwarp();                  // the stage has been read
        if (!TMA || lane == 0) copy_ahead();
        if (++stage == kQ4Stages) { stage = 0; parity ^= 1; }
      }
    }

    // All but one warp of the worker put their sums down; that one, another every time, adds them to its own.
    const int first_row = unit * kRows, last_row = min(kRows, p.n - first_row) - 1;
    auto each_sum = [&](auto&& f) {
#pragma unroll
      for (int rt = 0; rt < RT; ++rt)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int c = 0; c < 4; ++c) f((nt * 8 + t * 2 + c % 2) * kSumStride + rt * 16 + c / 2 * 8 + g, acc[rt][nt][c]);
    };
    const int adder = round % parts;
    if (mine) {
      if (parts > 1) {
        worker_barrier(local, parts);      // the sums before have been read
        if (part_of != adder) {
          float* to = sums + (part_of < adder ? part_of : part_of - 1) * kBuffer;
          each_sum([&](int at, float v) { to[at] = v; });
        }
        worker_barrier(local, parts);
      }
      if (part_of == adder) {
        for (int v = 0; v < parts - 1; ++v) each_sum([&](int at, float& a) { a += sums[v * kBuffer + at]; });
        each_sum([&](int at, float v) { sums[at] = v; });
      }
      if (p.slices == 1) {
        // the rows of X are shared out among the warps
        if (parts > 1) worker_barrier(local, parts);
        else __syncwarp();
        const int j = lane % kRows;
        if (j <= last_row)
          for (int r = part_of * (2 / RT) + lane / kRows; r < rows; r += parts * (2 / RT)) {
            float s = sums[r * kSumStride + j];
            if (columns != rows) s += sums[(r + rows) * kSumStride + j] + sums[(r + 2 * rows) * kSumStride + j];
            store_real(p.Y, (r0 + r) * p.ldy + first_row + j, p.type_y, s * (1 / kQ4Unit<BF16>));
          }
        __syncwarp();                        // the lanes' loops differ in length; what follows are barriers of whole warps
      }
    }
    if (p.slices > 1) {
      cluster_barrier();
      // this block's share of the outputs of its own units, from the sums of all blocks
      const int outputs = workers_here * rows * kRows;
      for (int at = slice * kThreads + tid; at < outputs; at += p.slices * kThreads) {
        const int j = at % kRows, r = at / kRows % rows, l = at / kRows / rows;
        const long long row = (worker_of(l) + static_cast<long long>(round) * workers) * kRows + j;
        if (row >= p.n) continue;
        const float* from = all_sums + l * buffers * kBuffer + r * kSumStride + j;
        float s = 0.0f;
        for (int v = 0; v < p.slices; ++v) {
          float rest = 0.0f;
          if (columns != rows) rest = load_cluster(from + rows * kSumStride, v) + load_cluster(from + 2 * rows * kSumStride, v);
          s += load_cluster(from, v) + rest;
        }
        store_real(p.Y, (r0 + r) * p.ldy + row, p.type_y, s * (1 / kQ4Unit<BF16>));
      }
      __syncwarp();                          // as above
      cluster_barrier();                     // no block writes its sums before all have read them
    }
  }
  if constexpr (!TMA) asm volatile("cp.async.wait_all;" ::: "memory");
}

}  // namespace cuasr_b200
