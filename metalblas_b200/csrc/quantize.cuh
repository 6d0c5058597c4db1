// Rows of floats to int8 rows with one fp32 scale each (symmetric, no zero
// point):
//
//   amax_r = max_c |x[r, c]|,  scale_r = amax_r / 127,
//   q[r, c] = rint(127 x[r, c] / amax_r)            (halves to even)
//
// The quotient is taken as 127 x over amax, not as x over the rounded scale, and
// 127 / amax is held as a sum hi + lo of two fp32 numbers, so that
// fma(x, hi, x lo) is the quotient rounded once to fp32.  For bf16 and fp16 x a
// quotient that is a half comes out exactly, and one that is not differs from the
// nearest half by more (2^-19 of it) than that rounding: q is the value of the
// real-number formula, halves included.  (For fp32 x the product y = 127 x rounds
// once, and hi + lo stands for 1 / amax.)
//
// A row of zeros has scale 0 and q 0.  A row that holds an infinity or a NaN
// has no scale: it gets scale NaN and q 0, so whatever is computed from it
// shows NaN.  |q| <= 127 always.
#pragma once
#include "mb_common.cuh"

#include <type_traits>

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

// Zeros all but the first n elements of v.
template <class T> __device__ __forceinline__ void keep_first(Vec<T> &v, int n) {
  if (n >= Vec<T>::V) return;
  uint32_t *w = &v.u.q.x;
  const int bytes = n * (int)sizeof(T);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int b = bytes - 4 * i;
    w[i] = b >= 4 ? w[i] : (b <= 0 ? 0u : w[i] & ((1u << (8 * b)) - 1));
  }
}

// 16 bytes that are read once, zeros where `on` is false.  As volatile assembly a
// batch of these is issued as written, ahead of its uses; left to itself the
// compiler interleaved loads and sums to save registers, two or three in flight
// (combine of 4096 tokens x 8 x 4096 bf16: 72 us, 4.2 TB/s).
// KEEP: the neighbouring thread reads the same word, so it stays in L1.
// The loads are ordinary (coherent) ones: a kernel launched with programmatic
// serialization may be resident while the kernel before it still writes these
// bytes, and pdl_wait orders ordinary loads only; the non-coherent form is for
// memory that nobody writes as long as the kernel lives.
template <bool KEEP = false>
__device__ __forceinline__ uint4 load_once(const void *p, bool on) {
  uint4 v;
  if constexpr (KEEP)
    asm volatile(
        "{\n\t.reg .pred q;\n\tsetp.ne.u32 q, %5, 0;\n\t"
        "mov.u32 %0, 0;\n\tmov.u32 %1, 0;\n\tmov.u32 %2, 0;\n\tmov.u32 %3, 0;\n\t"
        "@q ld.global.v4.u32 {%0, %1, %2, %3}, [%4];\n\t}"
        : "=&r"(v.x), "=&r"(v.y), "=&r"(v.z), "=&r"(v.w)
        : "l"(p), "r"((uint32_t)on));
  else
    asm volatile(
        "{\n\t.reg .pred q;\n\tsetp.ne.u32 q, %5, 0;\n\t"
        "mov.u32 %0, 0;\n\tmov.u32 %1, 0;\n\tmov.u32 %2, 0;\n\tmov.u32 %3, 0;\n\t"
        "@q ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];\n\t}"
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

// The largest |x| of a row, as ordered bits: NaN above infinity above every finite
// value, so an integer maximum never loses a NaN.  16-bit types are compared two
// to a word, as they come.
template <class T> struct MaxAbs {
  uint32_t m = 0;
  __device__ __forceinline__ void add(const Vec<T> &v) {
    const uint32_t w[4] = {v.u.q.x, v.u.q.y, v.u.q.z, v.u.q.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (sizeof(T) == 2) m = __vmaxu2(m, w[i] & 0x7fff7fffu);
      else m = max(m, w[i] & 0x7fffffffu);
    }
  }
  // As fp32 bits.
  __device__ __forceinline__ uint32_t bits() const {
    if constexpr (sizeof(T) == 2) {
      const uint32_t h = max(m & 0xffffu, m >> 16);
      if constexpr (std::is_same_v<T, __half>) return __float_as_uint(__half2float(__ushort_as_half((unsigned short)h)));
      return h << 16;
    }
    return m;
  }
};

// Two fp32 at a time: the same roundings as one by one.
__device__ __forceinline__ unsigned long long &bits64(float2 &v) { return reinterpret_cast<unsigned long long &>(v); }
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 o;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(bits64(o)) : "l"(bits64(a)), "l"(bits64(b)));
  return o;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 o;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(bits64(o)) : "l"(bits64(a)), "l"(bits64(b)));
  return o;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 o;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(bits64(o)) : "l"(bits64(a)), "l"(bits64(b)), "l"(bits64(c)));
  return o;
}

// How the elements of a row of T become integers.
template <class T> struct RowQuant {
  static constexpr bool kLong = sizeof(T) == 4;  // fp32: y = 127 x
  float hi, lo, pre;
  bool dead;  // zero or non-finite row: q = 0
  __device__ __forceinline__ explicit RowQuant(uint32_t bits) {
    constexpr float kTop = kLong ? 1.f : 127.f;
    const float m = __uint_as_float(bits);
    dead = bits == 0 || bits >= 0x7f800000u;
    // a row whose 127 x or 127 / amax would leave fp32's range (lo included) is
    // moved by a power of two first: exact, and the same for x and amax
    pre = m > 0x1p90f ? 0x1p-96f : (m < 0x1p-60f ? 0x1p80f : 1.f);
    const float amax = dead ? 1.f : m * pre;
    // an approximate quotient serves as hi: lo makes up for what it is off, to
    // 2^-42 of the sum (three IEEE divisions by every thread of a row were a
    // third of the kernel's instructions)
    hi = __fdividef(kTop, amax);
    lo = fmaf(-hi, amax, kTop) * (hi * (1.f / kTop));
  }
  __device__ static __forceinline__ float scale(uint32_t bits) {
    return bits >= 0x7f800000u ? __uint_as_float(0x7fc00000u) : __fdiv_rn(__uint_as_float(bits), 127.f);
  }
  // N elements at once.  Adding 1.5 * 2^23 rounds to an integer, halves to even,
  // and leaves it in the low bits.  No division and no branch per element: bf16
  // significands over each other give halves so often (every other group of 256
  // elements has one) that deciding them apart took two thirds of all
  // instructions (16384 x 8192 bf16: 204 a vector of eight, 119 us).
  template <int N>
  __device__ __forceinline__ void q(float (&x)[N], uint32_t (&out)[N / 4]) const {
    constexpr float kMagic = 12582912.f;
    if (pre != 1.f) {
#pragma unroll
      for (int i = 0; i < N; ++i) x[i] *= pre;
    }
    uint32_t r[N];
#pragma unroll
    for (int i = 0; i < N; i += 2) {
      float2 y = make_float2(x[i], x[i + 1]);
      if constexpr (kLong) y = mul2(y, make_float2(127.f, 127.f));
      const float2 t = fma2(y, make_float2(hi, hi), mul2(y, make_float2(lo, lo)));
      const float2 s = add2(t, make_float2(kMagic, kMagic));
      r[i] = __float_as_uint(s.x);
      r[i + 1] = __float_as_uint(s.y);
    }
#pragma unroll
    for (int i = 0; i < N / 4; ++i) {
      const uint32_t a = __byte_perm(r[4 * i], r[4 * i + 1], 0x0040);
      const uint32_t b = __byte_perm(r[4 * i + 2], r[4 * i + 3], 0x0040);
      out[i] = dead ? 0u : __byte_perm(a, b, 0x5410);
    }
  }
};

}  // namespace mb
