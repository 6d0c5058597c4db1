// Products with 4-bit weights (int4.cuh), one weight matrix or one per group of rows:
//
//   y[m, n] = sum_g s_e[n, g] (sum_{k in g} x[m, k] (u_e[n, k] - z_e[n, g])) + bias[n]
//
// for rows m of matrix e, offsets[e] <= m < offsets[e + 1]; rows at or past
// offsets[groups] are set to zero.  u - z is an integer of at most 255 and exact
// in bf16 and fp16, a product with it is exact in fp32, and the sum of a group is
// scaled in fp32: the weights are never rounded.
#pragma once
#include "int4.cuh"

namespace mb {
namespace i4 {

constexpr int kMaxGroups = 1024;

struct GemmArgs {
  const void *x;
  int64_t x_rs;
  int M, N, K, group_log2;
  const uint8_t *w;
  int64_t w_rs, w_e;
  const void *scale;
  int64_t s_rs, s_e;
  const uint8_t *zero;
  int64_t z_rs, z_e;
  const void *bias;
  int bias_f32, scale_f32;
  int groups;
  const int *offsets;   // null: one matrix
  void *out;
  int64_t out_rs;
};

// A scale as it lies in memory, and its value: apart, so that several can be on their way.
template <class T> __device__ __forceinline__ uint32_t scale_bits(const GemmArgs &a, int64_t i) {
  return a.scale_f32 ? static_cast<const uint32_t *>(a.scale)[i] : static_cast<const uint16_t *>(a.scale)[i];
}
template <class T> __device__ __forceinline__ float scale_of(const GemmArgs &a, uint32_t bits) {
  if (a.scale_f32) return __uint_as_float(bits);
  const uint16_t h = (uint16_t)bits;
  return to_f32(reinterpret_cast<const T &>(h));
}

template <class T> __device__ __forceinline__ float bias_at(const GemmArgs &a, int64_t n) {
  return a.bias_f32 ? static_cast<const float *>(a.bias)[n] : to_f32(static_cast<const T *>(a.bias)[n]);
}

// The groups' rows and units of `tokens` rows each: row0[e] and first_unit[e] for e <=
// groups, by the whole block; the number of units.  `scan` has a word per warp.  Offsets
// that are not ascending name no groups: every row comes out as zeros (and no count
// can leave the range that the host has checked).
__device__ __forceinline__ int unit_table(const GemmArgs &a, int tokens, int *first_unit, int *row0, int *scan) {
  const int G = a.groups, tid = threadIdx.x, threads = blockDim.x, lane = tid & 31, warp = tid >> 5;
  for (int e = tid; e <= G; e += threads) row0[e] = e ? min(max(a.offsets[e], 0), a.M) : 0;
  __syncthreads();
  int wrong = 0;
  for (int e = tid; e < G; e += threads) wrong |= row0[e + 1] < row0[e];
  if (__syncthreads_or(wrong)) {
    for (int e = tid; e <= G; e += threads) row0[e] = 0;
    __syncthreads();
  }
  // each thread sums `per` consecutive groups, then a scan over threads
  const int per = (G + threads - 1) / threads;
  const int e0 = min(G, tid * per), e1 = min(G, e0 + per);
  auto units_of = [&](int e) { return (row0[e + 1] - row0[e] + tokens - 1) / tokens; };
  int sum = 0;
  for (int e = e0; e < e1; ++e) sum += units_of(e);
  int upto = sum;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int o = __shfl_up_sync(0xffffffffu, upto, d);
    if (lane >= d) upto += o;
  }
  if (lane == 31) scan[warp] = upto;
  __syncthreads();
  int at = upto - sum;
  for (int w = 0; w < warp; ++w) at += scan[w];
  for (int e = e0; e < e1; ++e) {
    first_unit[e] = at;
    at += units_of(e);
  }
  if (tid == threads - 1) first_unit[G] = at;
  __syncthreads();
  return first_unit[G];
}
__device__ __forceinline__ int group_of_unit(const int *first_unit, int groups, int u) {
  int lo = 0, hi = groups;  // first_unit[lo] <= u < first_unit[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (first_unit[mid] <= u) lo = mid;
    else hi = mid;
  }
  return lo;
}

// Zeros for the rows from `first` on, shared out over the grid; thread `tid` of `threads`.
template <class T> __device__ __forceinline__ void zero_rest(const GemmArgs &a, int64_t first, int tid, int threads) {
  const int64_t n = (a.M - first) * (int64_t)a.N;
  for (int64_t i = (int64_t)blockIdx.x * threads + tid; i < n; i += (int64_t)gridDim.x * threads) {
    const int64_t m = i / a.N;
    static_cast<T *>(a.out)[(first + m) * a.out_rs + (i - m * a.N)] = Elem<T>::store(0.f);
  }
}

}  // namespace i4
}  // namespace mb
