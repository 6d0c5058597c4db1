// int8 products with a scale for each row of A and each column of B, one B per
// group of rows:
//
//   C[m, n] = (sum_k A[m, k] B_e[k, n]) scale_a[m] scale_b[e, n] + bias[n]
//
// for rows m of group e, i.e. offsets[e] <= m < offsets[e + 1]; rows at or past
// offsets[groups] are zero.  The sum is exact in 32-bit integers (K <= 131071);
// it is converted to fp32 once, multiplied by scale_a, then by scale_b.
#pragma once
#include "mb_common.cuh"

namespace mb {

struct ScaledParams {
  int64_t M, N, K;
  int groups;
  const int8_t *A, *B;
  void *C;
  int64_t a_rs, a_cs, b_rs, b_cs, sB, c_rs, c_cs;
  const float *scale_a, *scale_b;
  int64_t sa_s, sb_s, sb_g;
  const void *bias;
  int64_t bias_s;
  int bias_f32;
  const int *offsets;
};

template <class TO>
__global__ void __launch_bounds__(256) scaled_simple_kernel(const ScaledParams p) {
  __shared__ int8_t As[16][17], Bs[16][17];
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  pdl_trigger();
  pdl_wait();
  for (int e = 0; e <= p.groups; ++e) {
    // group `groups` stands for the rows that belong to none
    const int64_t lo = p.offsets ? min((int64_t)max(p.offsets[e], 0), p.M) : (e ? p.M : 0);
    const int64_t hi = (p.offsets && e < p.groups) ? min((int64_t)max(p.offsets[e + 1], 0), p.M) : p.M;
    const int64_t rt = (max(hi - lo, (int64_t)0) + 15) / 16, ct = (p.N + 15) / 16;
    for (int64_t tile = blockIdx.x; tile < rt * ct; tile += gridDim.x) {
      const int64_t m = lo + tile / ct * 16 + ty, n = tile % ct * 16 + tx;
      int acc = 0;
      if (e < p.groups) {
        const int8_t *B = p.B + e * p.sB;
        for (int64_t k0 = 0; k0 < p.K; k0 += 16) {
          As[ty][tx] = (m < hi && k0 + tx < p.K) ? p.A[m * p.a_rs + (k0 + tx) * p.a_cs] : 0;
          Bs[ty][tx] = (n < p.N && k0 + ty < p.K) ? B[(k0 + ty) * p.b_rs + n * p.b_cs] : 0;
          __syncthreads();
          for (int k = 0; k < 16; ++k) acc += (int)As[ty][k] * (int)Bs[k][tx];
          __syncthreads();
        }
      }
      if (m < hi && n < p.N) {
        float v = 0.f;
        if (e < p.groups) {
          v = __int2float_rn(acc) * p.scale_a[m * p.sa_s] * p.scale_b[e * p.sb_g + n * p.sb_s];
          if (p.bias)
            v += p.bias_f32 ? static_cast<const float *>(p.bias)[n * p.bias_s]
                            : Elem<TO>::load(static_cast<const TO *>(p.bias)[n * p.bias_s], false);
        }
        static_cast<TO *>(p.C)[m * p.c_rs + n * p.c_cs] = Elem<TO>::store(v);
      }
    }
  }
}

}  // namespace mb
