// The int8 product with scales (scaled_tc.cuh) for very few rows: a decode
// step's one or two tokens, or a few rows spread over experts.
//
// Such a product is one pass over the weights and nothing else, so the work is
// cut to put the same number of weight bytes on every SM: the weight rows to
// read are numbered through and shared out evenly over two blocks per SM, and a
// block's rows, as steps of 512 bytes, evenly over its warps; a warp runs
// through whole rows but for the first and the last of its share.  The
// tensor-core kernel hands out 128 channels at a time, which leaves 36 of 148
// SMs idle at N = 14336, and starts later (TMEM, pipeline).  Measured on B200,
// one row: K x N = 4096 x 14336 11.5 us against 13.8, 8192 x 28672 40.0
// (5.9 TB/s) against 45.8.  With four rows the dp4a work and the rows' reads from shared
// memory bind it (17.6 us against 14.6), so it takes two at most.
//
// By group (GROUPED) every row of A is a product of its own with its group's
// weights: a decode step's rows nearly always have an expert each, and rows that
// share one find its weights in L2.
//
// Rows of up to 2048 bytes leave most of a warp's eight loads unused, and a row's
// wait, sum and reduction follow one another.  So with more rows than warps a warp
// takes several whole rows at a time (ROWSTEPS: the 512-byte steps of a row): one
// row, K x N = 432 x 32768 3.8 us against 10.6, 1024 x 32768 5.9 against 12.0, 2048 x
// 8192 3.8 against 6.4; eight rows with an expert each, 512 x 8192 9.8 against 23.0.
//
// A lane multiplies its 16 weight bytes by dp4a with the rows of A, which lie in
// shared memory, padded with zeros to whole vectors.  A run's 32-bit sums are
// added into shared memory with integer atomics: the sum is exact, so their
// order does not matter.  The block then applies the scales in the tensor-core
// kernel's order; results have the same bits.
#pragma once
#include "quantize.cuh"
#include "scaled_tc.cuh"

namespace mb {
namespace sg {

constexpr int GEMV_ROWS = 2;          // rows of A, one weight matrix
constexpr int GEMV_GROUPED_ROWS = 8;  // rows of A, weights by group
constexpr int GEMV_THREADS = 512;
constexpr int GEMV_BLOCKS_PER_SM = 2;
constexpr int GEMV_BATCH = 8;         // 512-byte steps in flight per warp: 128 KB an SM

struct GemvArgs {
  const int8_t *A, *B;   // K contiguous, 16-byte aligned rows
  int64_t a_rs, b_rs, sB;
  int K;
  int max_rows;          // weight rows of a block, at most
};

// ROWSTEPS: 1, 2 or 4, rows of at most as many steps, taken whole; 0: any rows.
template <int MR, bool GROUPED, int ROWSTEPS, class TO>
__global__ void __launch_bounds__(GEMV_THREADS, GEMV_BLOCKS_PER_SM)
scaled_gemv_kernel(const __grid_constant__ SgParams p, const GemvArgs g) {
  static_assert(!GROUPED || MR == 1, "a row of A at a time");
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  const int vecs = (g.K + 15) / 16;
  const int staged = GROUPED ? p.M : MR;
  uint4 *xs = reinterpret_cast<uint4 *>(smem_raw);                // [staged][vecs]
  int *acc = reinterpret_cast<int *>(xs + (int64_t)staged * vecs);  // [max_rows][MR]
  __shared__ int group_of[GEMV_GROUPED_ROWS];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  constexpr int W = GEMV_THREADS / 32;
  const int per_row = (g.K + 511) / 512;

  // this block's weight rows and this warp's steps of them, for `total` rows in all
  int64_t r0 = 0;
  int rows = 0, row = 0, k = 0, left = 0;
  auto share = [&](int64_t total) {
    r0 = total * blockIdx.x / gridDim.x;
    rows = (int)(total * (blockIdx.x + 1) / gridDim.x - r0);
    if constexpr (ROWSTEPS > 0) {
      row = (int)((int64_t)rows * warp / W);
      left = (int)((int64_t)rows * (warp + 1) / W) - row;  // rows
      return;
    }
    const int64_t steps = (int64_t)rows * per_row;
    const int64_t s0 = steps * warp / W;
    left = (int)(steps * (warp + 1) / W - s0);
    row = (int)(s0 / per_row);
    k = (int)(s0 - (int64_t)row * per_row);
  };
  uint4 w[GEMV_BATCH];
  // steps k .. k+run-1 of the weight row at src, from step b of them
  auto fetch = [&](const int8_t *src, int run, int b) {
    const int v0 = (k + b) * 32 + lane, stop = min((k + run) * 32, vecs);
#pragma unroll
    for (int i = 0; i < GEMV_BATCH; ++i) w[i] = load_once(src + (int64_t)(v0 + i * 32) * 16, v0 + i * 32 < stop);
  };

  // whole rows: the next of them, `at` its A row, n its column
  int n = 0, at = 0;
  constexpr int RS = ROWSTEPS ? ROWSTEPS : 1, RB = GEMV_BATCH / RS;
  // (N is more than a batch: rows are taken whole when there are more than warps)
  auto fetch_rows = [&]() {
#pragma unroll
    for (int j = 0; j < RB; ++j) {
      const int wrap = GROUPED && n + j >= p.N;
      const int e = GROUPED && j < left ? min(group_of[at + wrap], p.groups - 1) : 0;
      const int8_t *src = g.B + (p.one_b ? 0 : e) * g.sB + (n + j - (wrap ? p.N : 0)) * g.b_rs;
#pragma unroll
      for (int i = 0; i < RS; ++i) w[j * RS + i] = load_once(src + (i * 32 + lane) * 16, j < left && i * 32 + lane < vecs);
    }
  };

  for (int i = tid; i < g.max_rows * MR; i += GEMV_THREADS) acc[i] = 0;
  if (tid < GEMV_GROUPED_ROWS) group_of[tid] = 0;
  if constexpr (!GROUPED) {
    // The weights' way into L2 may begin while the previous kernel ends.
    share(p.N);
    const int bytes = g.K & ~15;
    if (bytes)
      for (int i = tid; i < rows; i += GEMV_THREADS) prefetch_l2_bulk(g.B + (r0 + i) * g.b_rs, (uint32_t)bytes);
  }
  pdl_trigger();
  pdl_wait();
  if constexpr (!GROUPED) {
    n = (int)r0 + row;
    if constexpr (ROWSTEPS > 0) fetch_rows();
    else if (left > 0) fetch(g.B + n * g.b_rs, min(left, per_row - k), 0);
  }
  for (int i = tid; i < staged * vecs; i += GEMV_THREADS) {
    const int m = i / vecs, v = i - m * vecs;
    uint4 x = make_uint4(0, 0, 0, 0);
    if (m < p.M) {
      const int8_t *src = g.A + m * g.a_rs;
      if (v * 16 + 16 <= g.K) {
        x = *reinterpret_cast<const uint4 *>(src + v * 16);
      } else {
        int8_t b[16];
#pragma unroll
        for (int j = 0; j < 16; ++j) b[j] = v * 16 + j < g.K ? src[v * 16 + j] : 0;
        x = *reinterpret_cast<uint4 *>(b);
      }
    }
    xs[i] = x;
  }
  __syncthreads();
  int live = p.M;  // rows that belong to a group
  if constexpr (GROUPED) {
    // a row's group: the number of groups that end at or before it (p.groups: none)
    // (offsets that are not ascending: none for any row)
    int wrong = 0;
    for (int e = tid; e < p.groups; e += GEMV_THREADS) {
      const int end = p.offsets[e + 1];
      wrong |= e && min(max(end, 0), p.M) < min(max(p.offsets[e], 0), p.M);
      for (int m = 0; m < p.M; ++m)
        if (end <= m) atomicAdd(group_of + m, 1);
    }
    if (__syncthreads_or(wrong)) {
      if (tid < p.M) group_of[tid] = p.groups;
      __syncthreads();
    }
    while (live > 0 && group_of[live - 1] >= p.groups) --live;
    share((int64_t)live * p.N);
  }
  if constexpr (GROUPED) {
    const int64_t first = r0 + row;
    at = (int)(first / p.N);
    n = (int)(first - (int64_t)at * p.N);
  }
  bool fetched = !GROUPED;  // the first batch is on its way
  if constexpr (ROWSTEPS > 0) {
    while (left > 0) {
      if (!fetched) fetch_rows();
      fetched = false;
      int s[RB][MR];
#pragma unroll
      for (int j = 0; j < RB; ++j) {
#pragma unroll
        for (int m = 0; m < MR; ++m) s[j][m] = 0;
        const uint4 *x0 = xs + (GROUPED ? min(at + (n + j >= p.N), p.M - 1) * vecs : 0);
#pragma unroll
        for (int i = 0; i < RS; ++i) {
          const int v = min(i * 32 + lane, vecs - 1);
#pragma unroll
          for (int m = 0; m < MR; ++m) {
            const uint4 x = x0[m * vecs + v];
            s[j][m] = __dp4a((int)w[j * RS + i].x, (int)x.x, s[j][m]);
            s[j][m] = __dp4a((int)w[j * RS + i].y, (int)x.y, s[j][m]);
            s[j][m] = __dp4a((int)w[j * RS + i].z, (int)x.z, s[j][m]);
            s[j][m] = __dp4a((int)w[j * RS + i].w, (int)x.w, s[j][m]);
          }
        }
      }
#pragma unroll
      for (int j = 0; j < RB; ++j)
#pragma unroll
        for (int m = 0; m < MR; ++m) {
          const int sum = __reduce_add_sync(0xffffffffu, s[j][m]);
          if (lane == 0 && j < left) acc[(row + j) * MR + m] = sum;
        }
      left -= RB;
      row += RB;
      n += RB;
      if (GROUPED && n >= p.N) {
        n -= p.N;
        ++at;
      }
    }
  }
  while (ROWSTEPS == 0 && left > 0) {
    const int run = min(left, per_row - k);
    const int e = GROUPED ? min(group_of[at], p.groups - 1) : 0;
    const int8_t *src = g.B + (p.one_b ? 0 : e) * g.sB + n * g.b_rs;
    const uint4 *x0 = xs + (GROUPED ? (int64_t)at * vecs : 0);
    int s[MR];
#pragma unroll
    for (int m = 0; m < MR; ++m) s[m] = 0;
    for (int b = 0; b < run; b += GEMV_BATCH) {
      if (!fetched) fetch(src, run, b);
      fetched = false;
      const int v0 = (k + b) * 32 + lane;
#pragma unroll
      for (int i = 0; i < GEMV_BATCH; ++i) {
        const int v = min(v0 + i * 32, vecs - 1);  // past the end w is zero
#pragma unroll
        for (int m = 0; m < MR; ++m) {
          const uint4 x = x0[m * vecs + v];
          s[m] = __dp4a((int)w[i].x, (int)x.x, s[m]);
          s[m] = __dp4a((int)w[i].y, (int)x.y, s[m]);
          s[m] = __dp4a((int)w[i].z, (int)x.z, s[m]);
          s[m] = __dp4a((int)w[i].w, (int)x.w, s[m]);
        }
      }
    }
#pragma unroll
    for (int m = 0; m < MR; ++m) {
      const int sum = __reduce_add_sync(0xffffffffu, s[m]);
      if (lane == m) atomicAdd(acc + row * MR + m, sum);
    }
    left -= run;
    k = 0;
    ++row;
    if (++n == p.N && GROUPED) {
      n = 0;
      ++at;
    }
  }
  __syncthreads();
  TO *C = static_cast<TO *>(p.C);
  for (int i = tid; i < rows * MR; i += GEMV_THREADS) {
    int64_t m = i / rows, c = r0 + i - m * rows;  // rows of A outside, so that channels are stored in runs
    const int sum = acc[(i - (int)m * rows) * MR + (int)m];
    if constexpr (GROUPED) {
      m = c / p.N;
      c -= m * p.N;
    }
    if (m >= p.M) continue;
    const int e = GROUPED ? min(group_of[m], p.groups - 1) : 0;
    float v = scaled_sum(sum, p.scale_a[m * p.sa_s], p.scale_b[e * p.sb_g + c * p.sb_s]);
    if (p.bias) v = __fadd_rn(v, bias_at<TO>(p, c));
    C[m * p.c_rs + c * p.c_cs] = Elem<TO>::store(v);
  }
  // rows of no group
  for (int64_t m = live; m < p.M; ++m)
    for (int64_t c = (int64_t)blockIdx.x * GEMV_THREADS + tid; c < p.N; c += (int64_t)gridDim.x * GEMV_THREADS)
      C[m * p.c_rs + c * p.c_cs] = Elem<TO>::store(0.f);
}

// Two to sixteen rows, one weight matrix: the same single balanced pass, with the
// rows of A as the 16 rows of a warp-level int8 MMA and eight weight rows as its
// columns.  A lane loads 16 consecutive bytes of one weight row, which serve as
// the B words of two MMAs: the sum does not mind which bytes of K a position of
// the instruction stands for, as long as A's words, read from shared memory the
// same way, agree.  What counts here is that every SM reads the same bytes and
// starts at once: the tcgen05 kernel, which hands out 128 channels at a time and
// sets up TMEM and a pipeline first, takes 8.7 us for 4 x 4096 x 4096 against 6.0.
// Its eight-row reads stream at 4.5 TB/s, so products of more weights go there.
//
// A block's warps share K (KS slices) and pairs of eight weight rows.
constexpr int THIN_ROWS = 16;
constexpr int THIN_THREADS = 512;
constexpr int THIN_KS = 8;                                  // slices of K
constexpr int THIN_GS = THIN_THREADS / 32 / THIN_KS;        // warps that share out the pairs
// Rows of A in shared memory, an odd number of 64 bytes apart (no bank conflicts).
__host__ __device__ constexpr int thin_pitch(int K) { return (K + 127) / 128 * 128 + 64; }
// Sums of a row of A in shared memory, 8 words modulo 32 apart.
__host__ __device__ constexpr int thin_sums(int rows) { return (rows + 15) / 32 * 32 + 40; }

__device__ __forceinline__ void mma_s8(int (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// MANY: more than eight rows of A.
template <bool MANY, class TO>
__global__ void __launch_bounds__(THIN_THREADS, 2) scaled_thin_kernel(const __grid_constant__ SgParams p, const GemvArgs g) {
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  constexpr int STAGED = MANY ? 16 : 8, BATCH = 4;
  const int pitch = thin_pitch(g.K), vecs = (g.K + 15) / 16, chunks = (g.K + 63) / 64, sums = thin_sums(g.max_rows);
  uint8_t *xs = smem_raw;                                          // [STAGED][pitch]
  int *acc = reinterpret_cast<int *>(smem_raw + STAGED * pitch);   // [STAGED][sums]
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int64_t r0 = (int64_t)p.N * blockIdx.x / gridDim.x;
  const int rows = (int)((int64_t)p.N * (blockIdx.x + 1) / gridDim.x - r0);
  for (int i = tid; i < STAGED * sums; i += THIN_THREADS) acc[i] = 0;
  {
    const int bytes = g.K & ~15;
    if (bytes)
      for (int i = tid; i < rows; i += THIN_THREADS) prefetch_l2_bulk(g.B + (r0 + i) * g.b_rs, (uint32_t)bytes);
  }
  pdl_trigger();
  pdl_wait();
  const int ks = warp % THIN_KS, gs = warp / THIN_KS;
  const int c0 = ks * chunks / THIN_KS, c1 = (ks + 1) * chunks / THIN_KS;
  const int pairs = (rows + 15) / 16, wrow = lane >> 2, piece = lane & 3;
  uint4 w[2][BATCH];
  // chunks c .. c+BATCH-1 of both groups of a pair: this lane's row and 16 bytes
  auto fetch = [&](int pair, int c) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int row = pair * 16 + h * 8 + wrow;
      const int8_t *src = g.B + (r0 + row) * g.b_rs + piece * 16;
#pragma unroll
      for (int i = 0; i < BATCH; ++i)
        w[h][i] = load_once(src + (c + i) * 64, row < rows && c + i < c1 && (c + i) * 4 + piece < vecs);
    }
  };
  if (gs < pairs && c0 < c1) fetch(gs, c0);
  for (int i = tid; i < STAGED * (pitch / 16); i += THIN_THREADS) {
    const int m = i / (pitch / 16), v = i - m * (pitch / 16);
    uint4 x = make_uint4(0, 0, 0, 0);
    if (m < p.M && v < vecs) {
      const int8_t *src = g.A + m * g.a_rs;
      if (v * 16 + 16 <= g.K) {
        x = *reinterpret_cast<const uint4 *>(src + v * 16);
      } else {
        int8_t b[16];
#pragma unroll
        for (int j = 0; j < 16; ++j) b[j] = v * 16 + j < g.K ? src[v * 16 + j] : 0;
        x = *reinterpret_cast<uint4 *>(b);
      }
    }
    *reinterpret_cast<uint4 *>(xs + m * pitch + v * 16) = x;
  }
  __syncthreads();
  bool fetched = true;
  for (int pair = gs; pair < pairs; pair += THIN_GS) {
    int d[2][4] = {};
    for (int c = c0; c < c1; c += BATCH) {
      if (!fetched) fetch(pair, c);
      fetched = false;
#pragma unroll
      for (int i = 0; i < BATCH; ++i) {
        // past the slice w is zero; A's word is any that exists
        const uint8_t *x = xs + wrow * pitch + min(c + i, chunks - 1) * 64 + piece * 16;
        const uint4 lo = *reinterpret_cast<const uint4 *>(x);
        uint4 hi = make_uint4(0, 0, 0, 0);
        if constexpr (MANY) hi = *reinterpret_cast<const uint4 *>(x + 8 * pitch);
        const uint32_t a0[4] = {lo.x, hi.x, lo.y, hi.y}, a1[4] = {lo.z, hi.z, lo.w, hi.w};
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          mma_s8(d[h], a0, w[h][i].x, w[h][i].y);
          mma_s8(d[h], a1, w[h][i].z, w[h][i].w);
        }
      }
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      int *s = acc + wrow * sums + pair * 16 + h * 8 + piece * 2;
      atomicAdd(s, d[h][0]);
      atomicAdd(s + 1, d[h][1]);
      if constexpr (MANY) {
        atomicAdd(s + 8 * sums, d[h][2]);
        atomicAdd(s + 8 * sums + 1, d[h][3]);
      }
    }
  }
  __syncthreads();
  TO *C = static_cast<TO *>(p.C);
  for (int i = tid; i < p.M * rows; i += THIN_THREADS) {
    const int m = i / rows, row = i - m * rows;
    const int64_t n = r0 + row;
    float v = scaled_sum(acc[m * sums + row], p.scale_a[m * p.sa_s], p.scale_b[n * p.sb_s]);
    if (p.bias) v = __fadd_rn(v, bias_at<TO>(p, n));
    C[m * p.c_rs + n * p.c_cs] = Elem<TO>::store(v);
  }
}

}  // namespace sg
}  // namespace mb
