// Products of few tokens with 4-bit weights: one balanced pass over the weights on
// warp-level MMA.  What counts is the weights' bytes, so every SM reads the same
// number of weight rows and starts at once.
//
// A unit is up to 8 NT tokens of one matrix; the N weight rows of every unit,
// one unit after another, are cut into one range per block (row by row, not tile by
// tile: 97 rows on each SM, not 96 or 112).  Inside a block an item is 16 rows x 256
// columns (2 KB); the items of the range, column slices outside and row tiles
// inside, are cut into one run per warp.  So a warp keeps to one or two slices,
// whose tokens it holds in registers as MMA fragments while the weights stream by:
// tokens pass through no shared memory and are read once per block.  Each warp
// copies its items ahead into a ring of its own (cp.async, no barrier but the
// warp's), and adds its 16 x 8 NT sums of a tile to its own place in shared
// memory; at the end the warps' sums are added in order.  Results repeat bit for bit.
//
// m16n8k16 with weights as the rows.  A lane needs K positions in an order of the
// instruction's, but the sum does not mind which columns they stand for as long as
// weights and tokens agree: a lane takes whole 32-bit words (8 columns of a row),
// and its tokens' fragment is gathered to match.  (w & 0x000f000f) | 0x43004300 is
// the pair (128 + u0, 128 + u4) in bf16; subtracting 128 + z is exact.
#pragma once
#include "int4_gemm.cuh"

namespace mb {
namespace i4 {

constexpr int FEW_WARPS = 16;
constexpr int FEW_THREADS = FEW_WARPS * 32;
constexpr int FEW_SLICE = 256;              // columns of an item
constexpr int FEW_ITEM = 16 * FEW_SLICE / 2;  // its bytes
constexpr int FEW_STAGES = 4;
template <int NT> struct FewCfg {
  static constexpr int TILES = NT == 1 ? 10 : 5;   // row tiles of a block at a time
  static constexpr int RING = FEW_WARPS * FEW_STAGES * FEW_ITEM;
  static constexpr int SUMS = FEW_WARPS * TILES * NT * 512;
  static constexpr int smem(int groups) { return RING + SUMS + (2 * (groups + 1) + 32) * 4; }
  static_assert(RING + SUMS + (2 * (kMaxGroups + 1) + 32) * 4 <= 232448, "shared memory");
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void *src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

template <class T>
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same_v<T, __half>)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// What a row's zero point is to the decoding of its nibbles.
template <class T, bool ZERO> struct Decode;
template <bool ZERO> struct Decode<__nv_bfloat16, ZERO> {
  uint32_t z2;   // ZERO: (z, z)
  __device__ __forceinline__ explicit Decode(float z) {
    if constexpr (ZERO) {
      const uint32_t b = __float_as_uint(z) >> 16;   // z is a whole number up to 255
      z2 = b | (b << 16);
    }
  }
  // columns (0, 4), (1, 5), (2, 6), (3, 7) of a word
  __device__ __forceinline__ void operator()(uint32_t w, uint32_t (&o)[4]) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t v = ((w >> (4 * i)) & 0x000f000fu) | 0x43004300u;   // 128 + u
      __nv_bfloat162 x = reinterpret_cast<const __nv_bfloat162 &>(v);
      const uint32_t c = ZERO ? 0x43004300u : 0x43084308u;
      x = __hsub2(x, reinterpret_cast<const __nv_bfloat162 &>(c));
      if constexpr (ZERO) x = __hsub2(x, reinterpret_cast<const __nv_bfloat162 &>(z2));   // 128 + z may take nine bits
      o[i] = reinterpret_cast<uint32_t &>(x);
    }
  }
};
template <bool ZERO> struct Decode<__half, ZERO> {
  __half2 lo, hi;   // -(1024 + z), -(64 + z)
  __device__ __forceinline__ explicit Decode(float z) {
    if constexpr (!ZERO) z = 8.f;
    lo = __float2half2_rn(-(1024.f + z));
    hi = __float2half2_rn(-(64.f + z));
  }
  __device__ __forceinline__ void operator()(uint32_t w, uint32_t (&o)[4]) const {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint32_t s = w >> (8 * i);
      const uint32_t a = (s & 0x000f000fu) | 0x64006400u;   // 1024 + u
      const uint32_t b = (s & 0x00f000f0u) | 0x64006400u;   // 1024 + 16 u
      const __half2 x = __hadd2(reinterpret_cast<const __half2 &>(a), lo);
      const __half2 y = __hfma2(reinterpret_cast<const __half2 &>(b), __float2half2_rn(0.0625f), hi);
      o[2 * i] = reinterpret_cast<const uint32_t &>(x);
      o[2 * i + 1] = reinterpret_cast<const uint32_t &>(y);
    }
  }
};

// The 8 columns of a token from k on, as the pairs (0, 4), (1, 5), (2, 6), (3, 7); zeros past K.
template <class T>
__device__ __forceinline__ void token_pairs(const T *row, int k, int K, bool aligned, uint32_t (&o)[4]) {
  uint4 v = make_uint4(0, 0, 0, 0);
  if (aligned && k + 8 <= K) {
    v = *reinterpret_cast<const uint4 *>(row + k);
  } else {
    uint16_t t[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) t[i] = k + i < K ? reinterpret_cast<const uint16_t *>(row)[k + i] : 0;
    v = make_uint4(t[0] | t[1] << 16, t[2] | t[3] << 16, t[4] | t[5] << 16, t[6] | t[7] << 16);
  }
  o[0] = __byte_perm(v.x, v.z, 0x5410);
  o[1] = __byte_perm(v.x, v.z, 0x7632);
  o[2] = __byte_perm(v.y, v.w, 0x5410);
  o[3] = __byte_perm(v.y, v.w, 0x7632);
}

// LW: words that a lane takes of a row at a time, so that four lanes' words lie in
// one group (1: groups of 32 columns, 2: 64, 4: 128 and 256).
template <class T, int LW, int NT, bool ZERO>
__global__ void __launch_bounds__(FEW_THREADS, 1) int4_few_kernel(const __grid_constant__ GemmArgs a, int x_aligned) {
  using Cfg = FewCfg<NT>;
  constexpr int TOKENS = 8 * NT, SUB = 32 * LW, SUBS = FEW_SLICE / SUB;  // columns scaled together, and such in a slice
  constexpr int HELD = SUBS > 4 ? 2 : 1;                                 // scales of a row that a lane fetches
  extern __shared__ __align__(1024) uint8_t smem[];
  float *sums = reinterpret_cast<float *>(smem + Cfg::RING);
  int *first_unit = reinterpret_cast<int *>(smem + Cfg::RING + Cfg::SUMS);
  int *row0 = first_unit + a.groups + 1, *scan = row0 + a.groups + 1;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int g = lane >> 2, t4 = lane & 3;
  const int wrow = ((g & 1) << 2) | (g & 2) | (g >> 2);   // the weight row of MMA row g (shared-memory banks)
  const uint32_t ring = static_cast<uint32_t>(__cvta_generic_to_shared(smem)) + warp * (FEW_STAGES * FEW_ITEM);
  const int row_bytes = (a.K + 1) / 2, slices = (a.K + FEW_SLICE - 1) / FEW_SLICE;
  const int scales = (a.K + (1 << a.group_log2) - 1) >> a.group_log2;

  int units = (a.M + TOKENS - 1) / TOKENS;
  if (!a.offsets) {
    // this block's rows are known: as much of them as may matter starts its way into L2
    // (with one unit; more units' rows are the same ones again)
    const int64_t r0 = (int64_t)a.N * blockIdx.x / gridDim.x, rows = (int64_t)a.N * (blockIdx.x + 1) / gridDim.x - r0;
    const int bytes = (int)min((int64_t)row_bytes, (int64_t)(96 << 10) / max((int64_t)1, rows)) & ~15;
    if (bytes && units == 1)
      for (int i = tid; i < rows; i += FEW_THREADS) prefetch_l2_bulk(a.w + (r0 + i) * a.w_rs, (uint32_t)bytes);
    pdl_wait();
  } else {
    pdl_wait();
    units = unit_table(a, TOKENS, first_unit, row0, scan);
  }
  const int64_t total = (int64_t)units * a.N;
  int64_t at = total * blockIdx.x / gridDim.x;
  const int64_t end = total * (blockIdx.x + 1) / gridDim.x;

  while (at < end) {
    // up to TILES row tiles of one unit
    const int u = (int)(at / a.N), n0 = (int)(at - (int64_t)u * a.N);
    const int rows = (int)min(min(end - at, (int64_t)(a.N - n0)), (int64_t)(16 * Cfg::TILES));
    int e = 0, m0 = u * TOKENS, m1 = a.M;
    if (a.offsets) {
      e = group_of_unit(first_unit, a.groups, u);
      m0 = row0[e] + (u - first_unit[e]) * TOKENS;
      m1 = row0[e + 1];
    }
    m1 = min(m1, m0 + TOKENS);
    const int tiles = (rows + 15) / 16, items = slices * tiles;
    const int i0 = items * warp / FEW_WARPS, i1 = items * (warp + 1) / FEW_WARPS;
    const uint8_t *w = a.w + e * a.w_e + (int64_t)n0 * a.w_rs;

    // item i of the block to stage st of the ring: 128 bytes of 16 rows, a lane 16 bytes of
    // rows lane / 8, + 4, + 8, + 12; chunks are exchanged by row so that reads meet no bank twice
    const int crow = lane >> 3, chunk = lane & 7;
    int fs = i0 / tiles, ft = i0 - fs * tiles;   // the next item to fetch
    int fetched = i0;
    auto fetch = [&](int st) {
      if (fetched < i1) {
        const int off = fs * (FEW_SLICE / 2) + chunk * 16;
        const int bytes = min(max(row_bytes - off, 0), 16);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int r = crow + 4 * i, row = ft * 16 + r;
          const bool on = row < rows && bytes > 0;
          cp_async16(ring + st * FEW_ITEM + r * 128 + ((chunk ^ (r & 7)) << 4),
                     on ? w + (int64_t)row * a.w_rs + off : a.w, on ? bytes : 0);
        }
        ++fetched;
        if (++ft == tiles) { ft = 0; ++fs; }
      }
      cp_async_commit();
    };
#pragma unroll
    for (int st = 0; st < FEW_STAGES; ++st) fetch(st);

    // scales and zero points of the warp's next item: rows wrow and wrow + 8, sums t4 and t4 + 4
    float sc[2][HELD], zc[2][HELD];
    auto fetch_scales = [&](int s, int t) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int row = t * 16 + h * 8 + wrow;
#pragma unroll
        for (int j = 0; j < HELD; ++j) {
          const int q = (s * FEW_SLICE + (t4 + 4 * j) * SUB) >> a.group_log2;
          const bool on = row < rows && t4 + 4 * j < SUBS && q < scales;
          sc[h][j] = on ? scale_at<T>(a, e * a.s_e + (int64_t)(n0 + row) * a.s_rs + q) : 0.f;
          if constexpr (ZERO) zc[h][j] = on ? (float)a.zero[e * a.z_e + (int64_t)(n0 + row) * a.z_rs + q] : 0.f;
        }
      }
    };

    float *own = sums + (size_t)warp * (Cfg::TILES * NT * 128) + lane * 4;
    for (int i = 0; i < tiles * NT; ++i) *reinterpret_cast<float4 *>(own + i * 128) = make_float4(0.f, 0.f, 0.f, 0.f);

    uint32_t x[NT][8][4];
    int s = i0 / tiles, t = i0 - s * tiles, held = -1, st = 0;
    if (i0 < i1) fetch_scales(s, t);
    for (int i = i0; i < i1; ++i) {
      if (s != held) {
        held = s;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const int m = m0 + n * 8 + g;
          const T *row = static_cast<const T *>(a.x) + (int64_t)m * a.x_rs;
#pragma unroll
          for (int v = 0; v < 8; ++v) {
            const int k = s * FEW_SLICE + (v / LW) * SUB + t4 * (8 * LW) + (v % LW) * 8;
            if (m < m1) token_pairs(row, k, a.K, x_aligned, x[n][v]);
            else x[n][v][0] = x[n][v][1] = x[n][v][2] = x[n][v][3] = 0;
          }
        }
      }
      float sn[2][HELD], zn[2][HELD];
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int j = 0; j < HELD; ++j) {
          sn[h][j] = sc[h][j];
          if constexpr (ZERO) zn[h][j] = zc[h][j];
        }
      const int this_t = t;
      if (++t == tiles) { t = 0; ++s; }
      if (i + 1 < i1) fetch_scales(s, t);

      cp_async_wait<FEW_STAGES - 1>();
      __syncwarp();
      // this lane's words of rows wrow and wrow + 8
      uint32_t q[2][8];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint32_t base = ring + st * FEW_ITEM + (h * 8 + wrow) * 128;
#pragma unroll
        for (int j = 0; j < SUBS; ++j) {
          const int byte = j * (SUB / 2) + t4 * (4 * LW);
          const uint32_t p = base + ((((byte >> 4) ^ wrow) << 4) | (byte & 15));
          if constexpr (LW == 4)
            asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                         : "=r"(q[h][4 * j]), "=r"(q[h][4 * j + 1]), "=r"(q[h][4 * j + 2]), "=r"(q[h][4 * j + 3]) : "r"(p));
          else if constexpr (LW == 2)
            asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(q[h][2 * j]), "=r"(q[h][2 * j + 1]) : "r"(p));
          else
            asm volatile("ld.shared.u32 %0, [%1];" : "=r"(q[h][j]) : "r"(p));
        }
      }
      __syncwarp();
      fetch(st);
      if (++st == FEW_STAGES) st = 0;

      float acc[NT][4];
#pragma unroll
      for (int n = 0; n < NT; ++n) acc[n][0] = acc[n][1] = acc[n][2] = acc[n][3] = 0.f;
#pragma unroll
      for (int j = 0; j < SUBS; ++j) {
        const int src = (lane & ~3) | (j & 3);
        const float s0 = __shfl_sync(0xffffffffu, sn[0][j / 4], src), s1 = __shfl_sync(0xffffffffu, sn[1][j / 4], src);
        float z0 = 8.f, z1 = 8.f;
        if constexpr (ZERO) {
          z0 = __shfl_sync(0xffffffffu, zn[0][j / 4], src);
          z1 = __shfl_sync(0xffffffffu, zn[1][j / 4], src);
        }
        const Decode<T, ZERO> d0(z0), d1(z1);
        float d[NT][4];
#pragma unroll
        for (int n = 0; n < NT; ++n) d[n][0] = d[n][1] = d[n][2] = d[n][3] = 0.f;
#pragma unroll
        for (int v = j * LW; v < (j + 1) * LW; ++v) {
          uint32_t p0[4], p1[4];
          d0(q[0][v], p0);
          d1(q[1][v], p1);
#pragma unroll
          for (int h = 0; h < 4; h += 2) {
            const uint32_t f[4] = {p0[h], p1[h], p0[h + 1], p1[h + 1]};
#pragma unroll
            for (int n = 0; n < NT; ++n) mma16816<T>(d[n], f, x[n][v][h], x[n][v][h + 1]);
          }
        }
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          acc[n][0] = fmaf(d[n][0], s0, acc[n][0]);
          acc[n][1] = fmaf(d[n][1], s0, acc[n][1]);
          acc[n][2] = fmaf(d[n][2], s1, acc[n][2]);
          acc[n][3] = fmaf(d[n][3], s1, acc[n][3]);
        }
      }
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        float4 *o = reinterpret_cast<float4 *>(own + (this_t * NT + n) * 128);
        const float4 v = *o;
        *o = make_float4(v.x + acc[n][0], v.y + acc[n][1], v.z + acc[n][2], v.w + acc[n][3]);
      }
    }
    cp_async_wait<0>();
    if (end - at == rows) pdl_trigger();
    __syncthreads();
    // four results of a tile: rows r and r + 8, tokens c and c + 1
    for (int i = tid; i < tiles * NT * 32; i += FEW_THREADS) {
      const int l = i & 31, tn = i >> 5, tile = tn / NT, n = tn - tile * NT;
      float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int k = 0; k < FEW_WARPS; ++k) {
        const float4 v = *reinterpret_cast<const float4 *>(sums + (size_t)k * (Cfg::TILES * NT * 128) + tn * 128 + l * 4);
        y.x += v.x; y.y += v.y; y.z += v.z; y.w += v.w;
      }
      const int lg = l >> 2, r = tile * 16 + (((lg & 1) << 2) | (lg & 2) | (lg >> 2)), m = m0 + n * 8 + (l & 3) * 2;
      const float o[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const int row = r + (c >> 1) * 8, mm = m + (c & 1);
        if (row < rows && mm < m1) {
          float v = o[c];
          if (a.bias) v += bias_at<T>(a, n0 + row);
          static_cast<T *>(a.out)[(int64_t)mm * a.out_rs + n0 + row] = Elem<T>::store(v);
        }
      }
    }
    __syncthreads();
    at += rows;
  }
  if (a.offsets) zero_rest<T>(a, row0[a.groups], tid, FEW_THREADS);
}

}  // namespace i4
}  // namespace mb
