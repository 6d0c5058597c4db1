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
#include "pack.cuh"

namespace mb {

template <class T> __device__ __forceinline__ float to_f32(T v) { return Elem<T>::load(v, false); }

// 16 bytes of a row.
template <class T> struct Vec {
  static constexpr int V = 16 / (int)sizeof(T);
  union { uint4 q; T t[V]; } u;
  __device__ __forceinline__ Vec() {}
  __device__ __forceinline__ float f(int i) const { return to_f32(u.t[i]); }
  __device__ __forceinline__ void set(int i, float v) { u.t[i] = Elem<T>::store(v); }
  __device__ __forceinline__ void zero() { u.q = make_uint4(0, 0, 0, 0); }
};

// Elements c .. c+V-1 of a row of H, zeros outside it.  AL: rows start on 16
// bytes and c is a multiple of V.  Otherwise the 16 bytes are cut out of the
// one or two aligned words that hold them: the second word is read only when it
// holds some of them, so nothing past the row's last word is touched, and the
// neighbouring thread's copy of it comes from L1.
template <class T, bool AL>
__device__ __forceinline__ Vec<T> load_vec(const T *row, int c, int H) {
  constexpr int V = Vec<T>::V;
  Vec<T> v;
  if (c >= 0 && c + V <= H) {
    if constexpr (AL) {
      v.u.q = *reinterpret_cast<const uint4 *>(row + c);
    } else {
      const uintptr_t a = reinterpret_cast<uintptr_t>(row + c);
      const uint32_t off = (uint32_t)(a & 15);
      const uint4 *w = reinterpret_cast<const uint4 *>(a - off);
      v.u.q = w[0];
      if (off) v.u.q = bytes_at(v.u.q, w[1], off);
    }
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) v.u.t[i] = (c + i >= 0 && c + i < H) ? row[c + i] : Elem<T>::store(0.f);
  }
  return v;
}

// The first column of a row's vectors: 0 when the row starts on 16 bytes, else
// the column (<= 0) whose address does, so that whole vectors can be stored.
template <class T, bool AL> __device__ __forceinline__ int frame(const T *row) {
  if constexpr (AL) return 0;
  return -(int)((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(T));
}
// Store to c .. c+V-1 (c on the row's frame), the part inside the row only.
template <class T>
__device__ __forceinline__ void store_vec(T *row, int c, int H, const Vec<T> &v) {
  constexpr int V = Vec<T>::V;
  if (c >= 0 && c + V <= H) {
    *reinterpret_cast<uint4 *>(row + c) = v.u.q;
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (c + i >= 0 && c + i < H) row[c + i] = v.u.t[i];
  }
}

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
