// Rows of floats to int8 rows with one fp32 scale each (symmetric, no zero
// point):
//
//   amax_r = max_c |x[r, c]|,  scale_r = amax_r / 127,
//   q[r, c] = rint(127 x[r, c] / amax_r)            (halves to even)
//
// The quotient is taken as 127 x over amax, not as x over the rounded scale:
// for bf16 and fp16 the product 127 x is exact in fp32, and a quotient of two
// such numbers that is not a half differs from the nearest half by more than
// an fp32 rounding, so q is the value of the real-number formula, halves
// included.  (For fp32 x the product rounds once.)
//
// A row of zeros has scale 0 and q 0.  A row that holds an infinity or a NaN
// has no scale: it gets scale NaN and q 0, so whatever is computed from it
// shows NaN.  |q| <= 127 always.
#pragma once
#include "mb_common.cuh"

namespace mb {

template <class T> __device__ __forceinline__ float to_f32(T v) { return Elem<T>::load(v, false); }

// V consecutive elements: one 16-byte load, or one element.
template <class T, int V> struct Vec {
  static_assert(V * sizeof(T) == 16, "16-byte vectors");
  union { uint4 q; T t[V]; } u;
  __device__ __forceinline__ void load(const T *p) { u.q = *reinterpret_cast<const uint4 *>(p); }
  __device__ __forceinline__ void store(T *p) const { *reinterpret_cast<uint4 *>(p) = u.q; }
  __device__ __forceinline__ void zero() { u.q = make_uint4(0, 0, 0, 0); }
  __device__ __forceinline__ float f(int i) const { return to_f32(u.t[i]); }
  __device__ __forceinline__ void set(int i, float v) { u.t[i] = Elem<T>::store(v); }
};
template <class T> struct Vec<T, 1> {
  T t;
  __device__ __forceinline__ void load(const T *p) { t = *p; }
  __device__ __forceinline__ void store(T *p) const { *p = t; }
  __device__ __forceinline__ void zero() { t = Elem<T>::store(0.f); }
  __device__ __forceinline__ float f(int) const { return to_f32(t); }
  __device__ __forceinline__ void set(int, float v) { t = Elem<T>::store(v); }
};

// |x| of a row as ordered bits: NaN above infinity above every finite value,
// so an integer maximum never loses a NaN.
__device__ __forceinline__ uint32_t abs_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }

// How a row's elements become integers.
struct RowQuant {
  float amax, inv, pre, scale;
  bool dead;  // zero or non-finite row: q = 0
  __device__ __forceinline__ explicit RowQuant(uint32_t bits) {
    const float m = __uint_as_float(bits);
    dead = bits == 0 || bits >= 0x7f800000u;
    scale = bits >= 0x7f800000u ? __uint_as_float(0x7fc00000u) : __fdiv_rn(m, 127.f);
    // a row whose 127 x or 127 / amax would leave fp32's range is moved by a
    // power of two first (exact, and the same for x and amax)
    pre = m > 0x1p120f ? 0x1p-64f : (m < 0x1p-100f ? 0x1p64f : 1.f);
    amax = m * pre;
    inv = __fdiv_rn(127.f, amax);
  }
  __device__ __forceinline__ int q(float x) const {
    // x * inv is within 2e-5 of the quotient (two roundings of a value <= 127);
    // only a result that near to a half needs the quotient itself.
    x *= pre;
    const float t = x * inv;
    float r = rintf(t);
    if (fabsf(t - r) > 0.4999f) r = rintf(__fdiv_rn(x * 127.f, amax));
    return (int)r;
  }
};

}  // namespace mb
