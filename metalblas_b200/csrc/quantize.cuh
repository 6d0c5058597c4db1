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

// 16 bytes of a row.
template <class T> struct Vec {
  static constexpr int V = 16 / (int)sizeof(T);
  union { uint4 q; T t[V]; } u;
  __device__ __forceinline__ Vec() {}
  __device__ __forceinline__ float f(int i) const { return to_f32(u.t[i]); }
  __device__ __forceinline__ void set(int i, float v) { u.t[i] = Elem<T>::store(v); }
  __device__ __forceinline__ void zero() { u.q = make_uint4(0, 0, 0, 0); }
};

// 16 bytes starting `off` bytes into the 32 bytes a:b, without branches.
__device__ __forceinline__ uint4 cut16(const uint4 &a, const uint4 &b, uint32_t off) {
  const bool two = off & 8, one = off & 4;
  const uint32_t x0 = two ? a.z : a.x, x1 = two ? a.w : a.y, x2 = two ? b.x : a.z, x3 = two ? b.y : a.w,
                 x4 = two ? b.z : b.x, x5 = two ? b.w : b.y;
  const uint32_t y0 = one ? x1 : x0, y1 = one ? x2 : x1, y2 = one ? x3 : x2, y3 = one ? x4 : x3, y4 = one ? x5 : x4;
  const uint32_t sh = (off & 3) * 8;
  return make_uint4(__funnelshift_r(y0, y1, sh), __funnelshift_r(y1, y2, sh), __funnelshift_r(y2, y3, sh),
                    __funnelshift_r(y3, y4, sh));
}

// 16 bytes that are read once, zeros where `on` is false.  As volatile assembly a
// batch of these is issued as written, ahead of its uses; left to itself the
// compiler interleaved loads and sums to save registers, two or three in flight
// (combine of 4096 tokens x 8 x 4096 bf16: 72 us, 4.2 TB/s).
__device__ __forceinline__ uint4 load_once(const void *p, bool on) {
  uint4 v;
  asm volatile(
      "{\n\t.reg .pred q;\n\tsetp.ne.u32 q, %5, 0;\n\t"
      "mov.u32 %0, 0;\n\tmov.u32 %1, 0;\n\tmov.u32 %2, 0;\n\tmov.u32 %3, 0;\n\t"
      "@q ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];\n\t}"
      : "=&r"(v.x), "=&r"(v.y), "=&r"(v.z), "=&r"(v.w)
      : "l"(p), "r"((uint32_t)on));
  return v;
}

// The V elements at p.  AL: on a 16-byte boundary.  Otherwise they are cut out of
// the one or two aligned words that hold them: the second word is read only
// when it holds some of them, so no word without an element of the row is
// touched, and the neighbouring thread's copy of it comes from L1.
template <class T, bool AL>
__device__ __forceinline__ Vec<T> load16(const T *p) {
  Vec<T> v;
  if constexpr (AL) {
    v.u.q = *reinterpret_cast<const uint4 *>(p);
  } else {
    const uintptr_t a = reinterpret_cast<uintptr_t>(p);
    const uint32_t off = (uint32_t)(a & 15);
    const uint4 *w = reinterpret_cast<const uint4 *>(a - off);
    v.u.q = cut16(w[0], w[off ? 1 : 0], off);
  }
  return v;
}
// Elements c .. c+V-1 of a row of H, zeros outside it.
template <class T, bool AL>
__device__ __forceinline__ Vec<T> load_vec(const T *row, int c, int H) {
  constexpr int V = Vec<T>::V;
  if (c >= 0 && c + V <= H) return load16<T, AL>(row + c);
  Vec<T> v;
#pragma unroll
  for (int i = 0; i < V; ++i) v.u.t[i] = (c + i >= 0 && c + i < H) ? row[c + i] : Elem<T>::store(0.f);
  return v;
}

// The first column of a row's vectors: 0 when the row starts on 16 bytes, else
// the column (<= 0) whose address does, so that whole vectors can be stored.
template <class T, bool AL> __device__ __forceinline__ int frame(const T *row) {
  if constexpr (AL) return 0;
  return -(int)((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(T));
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
    amax = dead ? 1.f : m * pre;
    inv = dead ? 0.f : __fdiv_rn(127.f, amax);
  }
  // N elements at once.  x * inv is within 2e-5 of the quotient (two roundings
  // of a value of at most 127), so only a result that near to a half needs the
  // quotient itself: it is looked for once per N elements, and found for about
  // one element in 25000.  Adding 1.5 * 2^23 rounds to an integer, halves to
  // even, and leaves it in the low bits; conversions run at a quarter of that
  // rate or less, and bf16 rows were bound by them (2.6 TB/s at 16384 x 8192).
  template <int N>
  __device__ __forceinline__ void q(const float (&x)[N], uint32_t (&out)[N / 4]) const {
    constexpr float kMagic = 12582912.f;
    float r[N], worst = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float t = x[i] * pre * inv;
      r[i] = t + kMagic;
      worst = fmaxf(worst, fabsf(t - (r[i] - kMagic)));
    }
    if (worst > 0.49997f) {
#pragma unroll
      for (int i = 0; i < N; ++i) r[i] = __fdiv_rn(x[i] * pre * 127.f, amax) + kMagic;
    }
#pragma unroll
    for (int i = 0; i < N / 4; ++i) {
      const uint32_t lo = __byte_perm(__float_as_uint(r[4 * i]), __float_as_uint(r[4 * i + 1]), 0x0040);
      const uint32_t hi = __byte_perm(__float_as_uint(r[4 * i + 2]), __float_as_uint(r[4 * i + 3]), 0x0040);
      out[i] = dead ? 0u : __byte_perm(lo, hi, 0x5410);
    }
  }
};

}  // namespace mb
