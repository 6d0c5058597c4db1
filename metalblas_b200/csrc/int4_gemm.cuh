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

template <class T> __device__ __forceinline__ float scale_at(const GemmArgs &a, int64_t i) {
  return a.scale_f32 ? static_cast<const float *>(a.scale)[i] : to_f32(static_cast<const T *>(a.scale)[i]);
}

template <class T>
__global__ void __launch_bounds__(256) int4_simple_kernel(const GemmArgs a) {
  const int lane = threadIdx.x & 31;
  pdl_trigger();
  pdl_wait();
  bool wrong = false;
  if (a.offsets)
    for (int e = 0; e < a.groups; ++e) wrong |= min(max(a.offsets[e + 1], 0), a.M) < (e ? min(max(a.offsets[e], 0), a.M) : 0);
  const int64_t tasks = (int64_t)a.M * a.N;
  for (int64_t i = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); i < tasks; i += (int64_t)gridDim.x * 8) {
    const int64_t m = i / a.N, n = i - m * a.N;
    int e = 0;
    if (a.offsets) {
      if (wrong) e = a.groups;
      while (e < a.groups && m >= a.offsets[e + 1]) ++e;
    }
    T *dst = static_cast<T *>(a.out) + m * a.out_rs + n;
    if (a.offsets && e == a.groups) {
      if (lane == 0) *dst = Elem<T>::store(0.f);
      continue;
    }
    const T *x = static_cast<const T *>(a.x) + m * a.x_rs;
    const uint8_t *w = a.w + e * a.w_e + n * a.w_rs;
    float y = 0.f;
    for (int g = 0; g << a.group_log2 < a.K; ++g) {
      const float z = a.zero ? (float)a.zero[e * a.z_e + n * a.z_rs + g] : 8.f;
      float s = 0.f;
      const int k1 = min(a.K, (g + 1) << a.group_log2);
      for (int k = (g << a.group_log2) + lane; k < k1; k += 32)
        s = fmaf(to_f32(x[k]), (float)((w[k >> 1] >> (4 * (k & 1))) & 15) - z, s);
      y = fmaf(s, scale_at<T>(a, e * a.s_e + n * a.s_rs + g), y);
    }
#pragma unroll
    for (int d = 16; d; d >>= 1) y += __shfl_xor_sync(0xffffffffu, y, d);
    if (a.bias) y += a.bias_f32 ? static_cast<const float *>(a.bias)[n] : to_f32(static_cast<const T *>(a.bias)[n]);
    if (lane == 0) *dst = Elem<T>::store(y);
  }
}

}  // namespace i4
}  // namespace mb
