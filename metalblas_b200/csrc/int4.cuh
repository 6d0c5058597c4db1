// Weights of 4 bits with a scale, and with a zero point where one is given, for
// each group of G consecutive columns of a row (G = 32, 64, 128 or 256):
//
//   w[n, k] = (u[n, k] - z[n, k / G]) s[n, k / G],  u in 0..15, z = 8 without one.
//
// Two values to a byte, the even column in the low half; a row of K columns has
// (K + 1) / 2 bytes and (K + G - 1) / G scales.
//
// quantize: s = amax / 7 in fp32 and then in the scales' type, amax the largest |x| of
// the group, and u = 8 + rint(x / s), halves to even, within 1..15.  A group of zeros
// has scale 0, one with an infinity or a NaN scale NaN; both have u = 8.
//
// rint(x / s) is decided exactly, halves included.  16-bit x have so many of them that
// they are decided without a branch or a residual (Quant16 below); for fp32 x, and
// scales below the normal range, t = x (1 / s) is close enough that the half h
// nearest to it is the one next to the true quotient, and the sign of x - h s, which
// one fused multiply-add gives without error, says on which side of h that lies.
//
// A warp takes a row's spans of 256 columns, four at a time where there is work for every
// SM, so that as many loads are on their way as registers allow.  4096 x 14336 bf16 in
// groups of 128: quantize 36.7 us (floor 22.7: 117 MB read, 31 MB written; issue slots 71 % in
// use, the logic pipe 53 %, 44 % of the warps active), dequantize 26.6 us (5.6 TB/s).  fp32: 65.5
// and 60.7 us (floor 40.6), where a lane's 8 columns are 32 bytes in two accesses.
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

// Eight quotients of 16-bit x as the nibbles 8 + rint(x / s).
//
// x (hi + lo), hi + lo being the inverse of the scale to 2^-42, is the quotient
// rounded once to fp32.  With a scale of 16 bits too a quotient that is a half comes out
// exactly, and another one differs from it by more than that rounding.  A scale of
// fp32 is amax / 7 rounded: then 7 x / amax, which is a half or 2^-18.7 of it away from
// one at least (x and amax have 11 bits at most and lie within 4 binades where the
// quotient reaches 1/2), is taken instead and moved by 2^-21 of itself to the side
// that x / s lies on: all ties of a group go one way, the way that the scale was rounded.
struct Quant16 {
  float hi, lo;
  // num / den, and the way that quotients move
  __device__ __forceinline__ Quant16(float num, float den, float move) {
    const float h = __fdividef(num, den);
    hi = h;
    lo = fmaf(fmaf(-h, den, num), __fdividef(1.f, den), h * move);
  }
  __device__ __forceinline__ uint32_t operator()(const float (&x)[8]) const {
    constexpr float kMagic = 12582912.f;   // 1.5 * 2^23: adding it rounds to an integer
    const float2 h = make_float2(hi, hi), l = make_float2(lo, lo), m = make_float2(kMagic, kMagic), n = make_float2(-kMagic, -kMagic);
    float2 q[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 v = make_float2(x[i], x[i + 4]);
      q[i] = add2(add2(fma2(v, h, mul2(v, l)), m), n);
    }
    // four nibbles are a whole number below 2^16
    float2 f = fma2(q[1], make_float2(16.f, 16.f), q[0]);
    f = fma2(q[2], make_float2(256.f, 256.f), f);
    f = fma2(q[3], make_float2(4096.f, 4096.f), f);
    f = add2(f, make_float2(kMagic + 34952.f, kMagic + 34952.f));   // 8 in each
    return __byte_perm(__float_as_uint(f.x), __float_as_uint(f.y), 0x5410);
  }
};

// A group's scale as it is stored, and what its columns are divided with.
template <class T, class S> struct GroupScale {
  S stored;
  float s0;       // its value
  Quant16 quant;  // of 16-bit x, where `direct`
  bool direct;
  __device__ __forceinline__ explicit GroupScale(uint32_t amax_bits) : quant(0.f, 1.f, 0.f) {
    const float amax = __uint_as_float(amax_bits);
    const float exact7 = __fdiv_rn(amax, 7.f);
    stored = Elem<S>::store(amax_bits < 0x7f800000u ? exact7 : __uint_as_float(0x7fc00000u));
    s0 = to_f32(stored);
    constexpr bool F32 = sizeof(S) == 4;
    // (scales of fp16 are normal numbers from 2^-14 on)
    direct = sizeof(T) == 2 && s0 >= (std::is_same_v<S, __half> ? 0x1p-14f : 0x1p-100f) && s0 < 0x1p100f;
    if constexpr (sizeof(T) == 2) {
      // x / s lies above 7 x / amax where s was rounded down: s - amax / 7 has the sign of 7 s - amax
      const float over = F32 ? fmaf(7.f, s0, -amax) : 0.f;
      const float move = over == 0.f ? 0.f : copysignf(0x1p-21f, -over);
      quant = Quant16(F32 ? 7.f : 1.f, F32 ? amax : s0, move);
    }
  }
};
// The nibbles of 8 columns by a scale of any kind.
template <class T> __device__ __forceinline__ uint32_t nibbles(const float (&x)[8], float s0) {
  if (!(s0 < INFINITY) || s0 == 0.f) return 0x88888888u;   // NaN, infinite, 0
  // groups of tiny values are moved by a power of two, so that 1 / s and h s stay in range
  const float pre = s0 < 0x1p-90f ? 0x1p100f : 1.f, s = s0 * pre, inv = __fdividef(1.f, s);
  uint32_t word = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float q = fminf(fmaxf(rounded_quotient(x[i] * pre, s, inv), -7.f), 7.f);   // (a scale that rounded down to a subnormal)
    word |= (uint32_t)((int)q + 8) << (4 * i);
  }
  return word;
}

// A lane takes 8 consecutive columns at a time, so a group has G / 8 neighbouring lanes
// and a warp 256 columns of one row, a span.  A task is B spans next to one another.  Of four
// spans each lane reduces and divides for one, lane & 3, and the others get it from there
// (with every lane at work on all four, 4096 x 14336 took 44.7 us in bf16 and 73.2 in fp32, now 36.8
// and 65.5).  Rows off 16 bytes keep each lane's own columns: a column a lane with a warp's maximum
// for every 32 was slower, 15.6 us for 1001 x 4099 fp32 instead of 13.7.
template <class T, class S, bool AL, int B>
__global__ void __launch_bounds__(256) quantize_int4_kernel(const ConvertArgs a) {
  static_assert(B == 1 || B == 4, "spans");
  const int lane = threadIdx.x & 31, lanes = (1 << a.group_log2) / 8;   // of a group
  const uint32_t per_row = (a.cols + 256 * B - 1) / (256 * B);
  const int64_t tasks = a.rows * (int64_t)per_row;
  pdl_trigger();
  pdl_wait();
  constexpr int V = Vec<T>::V, NV = 8 / V;
  for (int64_t w = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); w < tasks; w += (int64_t)gridDim.x * 8) {
    const int64_t r = tasks < (1ll << 32) ? (uint32_t)w / per_row : w / per_row;
    const int cw = (int)(w - r * per_row) * (256 * B), c0 = cw + lane * 8;
    const T *src = static_cast<const T *>(a.src) + r * a.ld_src;
    Vec<T> v[B][NV];
#pragma unroll
    for (int b = 0; b < B; ++b)
#pragma unroll
      for (int i = 0; i < NV; ++i) v[b][i] = load_vec<T, AL>(src, c0 + b * 256 + i * V, a.cols);
    uint8_t *row = static_cast<uint8_t *>(a.dst) + r * a.ld_dst;
    const bool words = (reinterpret_cast<uintptr_t>(row) & 3) == 0;
    uint32_t m[B];
#pragma unroll
    for (int b = 0; b < B; ++b) {
      MaxAbs<T> most;
#pragma unroll
      for (int i = 0; i < NV; ++i) most.add(v[b][i]);
      m[b] = most.bits();
    }
    uint32_t bits = m[0];
    if constexpr (B == 4) {
      const bool o1 = lane & 1, o2 = lane & 2;
      const uint32_t m0 = max(o1 ? m[1] : m[0], __shfl_xor_sync(0xffffffffu, o1 ? m[0] : m[1], 1));   // span lane & 1
      const uint32_t m2 = max(o1 ? m[3] : m[2], __shfl_xor_sync(0xffffffffu, o1 ? m[2] : m[3], 1));   // and 2 on
      bits = max(o2 ? m2 : m0, __shfl_xor_sync(0xffffffffu, o2 ? m0 : m2, 2));
    }
    for (int d = B; d < lanes; d <<= 1) bits = max(bits, __shfl_xor_sync(0xffffffffu, bits, d));
    const GroupScale<T, S> g(bits);
    const int own = cw + (lane & (B - 1)) * 256 + (lane & -lanes) * 8;   // the group's first column
    if ((lane & (lanes - 1)) < B && own < a.cols)
      static_cast<S *>(a.scale)[r * a.ld_scale + (own >> a.group_log2)] = g.stored;
    const bool all = __all_sync(0xffffffffu, g.direct || own >= a.cols);
#pragma unroll
    for (int b = 0; b < B; ++b) {
      const int c = c0 + b * 256, from = (lane & ~3) | b;
      if (cw + b * 256 >= a.cols) break;
      float x[8];
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int j = 0; j < V; ++j) x[i * V + j] = v[b][i].f(j);
      uint32_t word;
      Quant16 q = g.quant;
      if constexpr (B == 4 && sizeof(T) == 2) {
        q.hi = __shfl_sync(0xffffffffu, q.hi, from);
        q.lo = __shfl_sync(0xffffffffu, q.lo, from);
      }
      if (sizeof(T) == 2 && all) {
        word = q(x);
      } else {
        const float s0 = B == 4 ? __shfl_sync(0xffffffffu, g.s0, from) : g.s0;
        const bool direct = B == 4 ? __shfl_sync(0xffffffffu, (int)g.direct, from) : g.direct;
        word = direct ? q(x) : nibbles<T>(x, s0);
      }
      if (c >= a.cols) continue;
      if (words && c + 7 <= a.cols) {
        *reinterpret_cast<uint32_t *>(row + c / 2) = word;
      } else {
        for (int i = 0; i < (min(8, a.cols - c) + 1) / 2; ++i) row[c / 2 + i] = (uint8_t)(word >> (8 * i));
      }
    }
  }
}

template <class T, class S, bool AL, int B>
__global__ void __launch_bounds__(256) dequantize_int4_kernel(const ConvertArgs a) {
  const int lane = threadIdx.x & 31;
  const uint32_t per_row = (a.cols + 256 * B - 1) / (256 * B);
  const int64_t tasks = a.rows * (int64_t)per_row;
  pdl_trigger();
  pdl_wait();
  for (int64_t w = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); w < tasks; w += (int64_t)gridDim.x * 8) {
    const int64_t r = tasks < (1ll << 32) ? (uint32_t)w / per_row : w / per_row;
    const int c0 = (int)(w - r * per_row) * (256 * B) + lane * 8;
    const uint8_t *row = static_cast<const uint8_t *>(a.src) + r * a.ld_src;
    const S *scales = static_cast<const S *>(a.scale) + r * a.ld_scale;
    const bool words = (reinterpret_cast<uintptr_t>(row) & 3) == 0;
    uint32_t word[B], zero[B];
    S scale[B];
#pragma unroll
    for (int b = 0; b < B; ++b) {
      const int c = c0 + b * 256;
      word[b] = 0;
      zero[b] = 8;
      scale[b] = S();
      if (c >= a.cols) continue;
      if (words && c + 7 <= a.cols) {
        word[b] = *reinterpret_cast<const uint32_t *>(row + c / 2);
      } else {
        for (int i = 0; i < (min(8, a.cols - c) + 1) / 2; ++i) word[b] |= (uint32_t)row[c / 2 + i] << (8 * i);
      }
      scale[b] = scales[c >> a.group_log2];
      if (a.zero) zero[b] = a.zero[r * a.ld_zero + (c >> a.group_log2)];
    }
    T *out = static_cast<T *>(a.dst) + r * a.ld_dst;
#pragma unroll
    for (int b = 0; b < B; ++b) {
      const int c = c0 + b * 256, n = min(8, a.cols - c);
      if constexpr (!AL) {
        // Rows off 16 bytes leave a column a lane, 32 next to one another: the words of the
        // lanes that hold them by shuffles (1001 x 4099 fp32 24.9 us with each lane's own columns).
        const float own = to_f32(scale[b]);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int from = 4 * i + (lane >> 3), col = c - lane * 8 + 32 * i + lane;
          const uint32_t u = __shfl_sync(0xffffffffu, word[b], from) >> (4 * (lane & 7)) & 15;
          const float z = (float)__shfl_sync(0xffffffffu, zero[b], from), s = __shfl_sync(0xffffffffu, own, from);
          if (col < a.cols) out[col] = Elem<T>::store(((float)u - z) * s);
        }
        continue;
      }
      if (n <= 0) break;
      const float s = to_f32(scale[b]);
      const float2 s2 = make_float2(s, s);
      const float off = -(8388608.f + (float)zero[b]);   // 2^23 + u - (2^23 + z)
      const float2 o2 = make_float2(off, off);
      constexpr int V = Vec<T>::V;
#pragma unroll
      for (int i = 0; i < 8; i += V) {
        Vec<T> v;
#pragma unroll
        for (int j = 0; j < V; j += 2) {
          const uint32_t u = word[b] >> (4 * (i + j));
          const float2 f = make_float2(__uint_as_float((u & 15) | 0x4b000000u), __uint_as_float(((u >> 4) & 15) | 0x4b000000u));
          const float2 y = mul2(add2(f, o2), s2);
          v.set(j, y.x);
          v.set(j + 1, y.y);
        }
        if (n >= i + V) {
          *reinterpret_cast<uint4 *>(out + c + i) = v.u.q;
        } else {
#pragma unroll
          for (int j = 0; j < V; ++j)
            if (i + j < n) out[c + i + j] = v.u.t[j];
        }
      }
    }
  }
}

}  // namespace i4
}  // namespace mb
