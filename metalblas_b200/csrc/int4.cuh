// Weights of 4 bits with a scale, and with a zero point where one is given, for
// each group of G consecutive columns of a row (G = 32, 64, 128 or 256):
//
//   w[n, k] = (u[n, k] - z[n, k / G]) s[n, k / G],  u in 0..15, z = 8 without one.
//
// Two values to a byte, the even column in the low half; a row of K columns has
// (K + 1) / 2 bytes and (K + G - 1) / G scales.
//
// quantize: s = amax / 7 rounded to the scales' type, amax the largest |x| of the
// group, and u = 8 + rint(x / s), halves to even, within 1..15.  A group of zeros
// has scale 0, one with an infinity or a NaN scale NaN; both have u = 8.
//
// rint(x / s) is decided exactly: t = x (1 / s) is close enough that the half h
// nearest to it is the one next to the true quotient, and the sign of x - h s, which
// one fused multiply-add gives without error, says on which side of h that lies.
#pragma once
#include "mb_common.cuh"
#include "quantize.cuh"

namespace mb {
namespace i4 {

struct ConvertArgs {
  const void *src;      // quantize: rows of floats; dequantize: packed rows
  int64_t ld_src;
  void *dst;
  int64_t ld_dst;
  int64_t rows;
  int cols, group_log2;
  void *scale;          // [rows, groups]
  int64_t ld_scale;
  const uint8_t *zero;  // [rows, groups] or null
  int64_t ld_zero;
};

// x / s to the nearest integer, halves to even, for |x / s| < 2^20.
__device__ __forceinline__ float rounded_quotient(float x, float s, float inv) {
  constexpr float kMagic = 12582912.f;                   // 1.5 * 2^23: adding it rounds to an integer
  const float t = x * inv;
  const float n = __fsub_rn(__fadd_rn(t, kMagic), kMagic);
  const float h = n + copysignf(0.5f, t - n);            // the half nearest to t
  const float e = fmaf(-h, s, x);                        // its sign is that of x / s - h
  const float y = e == 0.f ? h : h + copysignf(0.25f, e);
  return __fsub_rn(__fadd_rn(y, kMagic), kMagic);
}

// A lane takes 8 consecutive columns, so a group has G / 8 neighbouring lanes and a
// warp 256 columns of one row.
template <class T, class S, bool AL>
__global__ void __launch_bounds__(256) quantize_int4_kernel(const ConvertArgs a) {
  const int lane = threadIdx.x & 31;
  const int64_t per_row = (a.cols + 255) / 256, tasks = a.rows * per_row;
  pdl_trigger();
  pdl_wait();
  for (int64_t w = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); w < tasks; w += (int64_t)gridDim.x * 8) {
    const int64_t r = w / per_row;
    const int c = (int)(w - r * per_row) * 256 + lane * 8;
    const T *row = static_cast<const T *>(a.src) + r * a.ld_src;
    constexpr int V = Vec<T>::V;
    float x[8];
    MaxAbs<T> m;
#pragma unroll
    for (int i = 0; i < 8; i += V) {
      const Vec<T> v = load_vec<T, AL>(row, c + i, a.cols);
      m.add(v);
#pragma unroll
      for (int j = 0; j < V; ++j) x[i + j] = v.f(j);
    }
    uint32_t bits = m.bits();
    for (int d = 1; d < (1 << a.group_log2) / 8; d <<= 1) bits = max(bits, __shfl_xor_sync(0xffffffffu, bits, d));
    // the scale as it is stored
    const bool finite = bits < 0x7f800000u;
    const S stored = Elem<S>::store(finite ? __fdiv_rn(__uint_as_float(bits), 7.f) : __uint_as_float(0x7fc00000u));
    const float s0 = to_f32(stored);
    if (c < a.cols && (c & ((1 << a.group_log2) - 1)) == 0)
      static_cast<S *>(a.scale)[r * a.ld_scale + (c >> a.group_log2)] = stored;
    // groups of tiny values are moved by a power of two, so that 1 / s and h s stay in range
    const float pre = s0 < 0x1p-90f ? 0x1p100f : 1.f, s = s0 * pre;
    const float inv = __fdividef(1.f, s);
    uint32_t word = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float q = rounded_quotient(x[i] * pre, s, inv);
      q = fminf(fmaxf(q, -7.f), 7.f);   // a scale that rounded down to a subnormal
      const uint32_t u = !finite || s0 == 0.f ? 8u : (uint32_t)((int)q + 8);
      word |= u << (4 * i);
    }
    if (c >= a.cols) continue;
    uint8_t *dst = static_cast<uint8_t *>(a.dst) + r * a.ld_dst + c / 2;
    const int bytes = (min(8, a.cols - c) + 1) / 2;
    if (bytes == 4 && (reinterpret_cast<uintptr_t>(dst) & 3) == 0) {
      *reinterpret_cast<uint32_t *>(dst) = word;
    } else {
      for (int i = 0; i < bytes; ++i) dst[i] = (uint8_t)(word >> (8 * i));
    }
  }
}

template <class T, class S, bool AL>
__global__ void __launch_bounds__(256) dequantize_int4_kernel(const ConvertArgs a) {
  const int lane = threadIdx.x & 31;
  const int64_t per_row = (a.cols + 255) / 256, tasks = a.rows * per_row;
  pdl_trigger();
  pdl_wait();
  for (int64_t w = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); w < tasks; w += (int64_t)gridDim.x * 8) {
    const int64_t r = w / per_row;
    const int c = (int)(w - r * per_row) * 256 + lane * 8;
    if (c >= a.cols) continue;
    const uint8_t *src = static_cast<const uint8_t *>(a.src) + r * a.ld_src + c / 2;
    const int n = min(8, a.cols - c);
    uint32_t word = 0;
    if (n >= 7 && (reinterpret_cast<uintptr_t>(src) & 3) == 0) {
      word = *reinterpret_cast<const uint32_t *>(src);
    } else {
      for (int i = 0; i < (n + 1) / 2; ++i) word |= (uint32_t)src[i] << (8 * i);
    }
    const int g = c >> a.group_log2;
    const float s = to_f32(static_cast<const S *>(a.scale)[r * a.ld_scale + g]);
    const float z = a.zero ? (float)a.zero[r * a.ld_zero + g] : 8.f;
    T *dst = static_cast<T *>(a.dst) + r * a.ld_dst + c;
    constexpr int V = Vec<T>::V;
#pragma unroll
    for (int i = 0; i < 8; i += V) {
      Vec<T> v;
#pragma unroll
      for (int j = 0; j < V; ++j) v.set(j, ((float)((word >> (4 * (i + j))) & 15) - z) * s);
      if (AL && n >= i + V) {
        *reinterpret_cast<uint4 *>(dst + i) = v.u.q;
      } else {
#pragma unroll
        for (int j = 0; j < V; ++j)
          if (i + j < n) dst[i + j] = v.u.t[j];
      }
    }
  }
}

}  // namespace i4
}  // namespace mb
