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
// has its items brought into a ring of its own by TMA (one lane issues, no barrier but
// the warp's), and adds its 16 x 8 NT sums of a tile to its own place in shared
// memory; at the end the warps' sums are added in order.  Results repeat bit for bit.
// The rows' scales lie in shared memory as fp32: loaded item by item, even one item
// ahead, they were a third of the time (1 x 4096 x 14336: 22.1 us, 13.9 without them).
//
// m16n8k16 with weights as the rows.  A lane needs K positions in an order of the
// instruction's, but the sum does not mind which columns they stand for as long as
// weights and tokens agree: a lane takes whole 32-bit words (8 columns of a row),
// and its tokens' fragment is gathered to match.  (w & 0x000f000f) | 0x43004300 is
// the pair (128 + u0, 128 + u4) in bf16; subtracting 128 + z is exact.
//
// 1 x 4096 x 14336: 15.2 us (floor 4.6, the weights at the copy's rate), 16 rows 21.8.
// Some 5 us are the start, the scales and the sums' end.  DRAM 30 MB, each weight once; no
// pipe is full (logic 50 % in use over the launch, issue slots 49 %, 19 % of the warps active).
// A lane's word of 8 weights takes 35 instructions (8.1 M for 229,376 of a warp), of which
// its decoding and MMA are 12; the others have not been counted.
#pragma once
#include "int4_gemm.cuh"
#include "tc_gemm.cuh"

namespace mb {
namespace i4 {

constexpr int FEW_SLICE = 256;                // columns of an item
constexpr int FEW_ITEM = 16 * FEW_SLICE / 2;  // its bytes
template <int NT> struct FewCfg {
    static constexpr int WARPS = NT == 1 ? 12 : 8;   // (two fragments of tokens take 64 registers)
  static constexpr int THREADS = WARPS * 32;
  static constexpr int STAGES = 48 / WARPS;
  static constexpr int TILES = 7;                  // row tiles of a block at a time
  static constexpr int RING = WARPS * STAGES * FEW_ITEM;
  static constexpr int SUMS = WARPS * TILES * NT * 512;
  static constexpr int SCALES = 15360;             // fp32 words of scales (and zero points)
  static constexpr int BARS = (WARPS * STAGES + 1) * 8;
  static constexpr int smem(int groups) { return 1024 + RING + SUMS + SCALES * 4 + BARS + (2 * (groups + 1) + 32) * 4; }
  static_assert(1024 + RING + SUMS + SCALES * 4 + BARS + (2 * (kMaxGroups + 1) + 32) * 4 <= 232448, "shared memory");
};

template <class T>
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same_v<T, __half>)
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// One lane of the warp, the same at every call.
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred q;\n\telect.sync _|q, 0xffffffff;\n\tselp.u32 %0, 1, 0, q;\n\t}" : "=r"(p));
  return p != 0;
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

// 8 columns of a token as the pairs (0, 4), (1, 5), (2, 6), (3, 7).
__device__ __forceinline__ void token_pairs(const uint4 &v, uint32_t (&o)[4]) {
  o[0] = __byte_perm(v.x, v.z, 0x5410);
  o[1] = __byte_perm(v.x, v.z, 0x7632);
  o[2] = __byte_perm(v.y, v.w, 0x5410);
  o[3] = __byte_perm(v.y, v.w, 0x7632);
}

// LW: words that a lane takes of a row at a time, so that four lanes' words lie in
// one group (1: groups of 32 columns, 2: 64, 4: 128 and 256).
template <class T, int LW, int NT, bool ZERO>
__global__ void __launch_bounds__(FewCfg<NT>::THREADS, 1)
    int4_few_kernel(const __grid_constant__ GemmArgs a, const __grid_constant__ CUtensorMap weights,
                    unsigned long long timeout_ns) {
  using Cfg = FewCfg<NT>;
  constexpr int TOKENS = 8 * NT, SUB = 32 * LW, SUBS = FEW_SLICE / SUB;  // columns scaled together, and such in a slice
  constexpr int WORDS = ZERO ? 2 : 1;                                    // a scale, or a scale and a zero point
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  float *sums = reinterpret_cast<float *>(smem + Cfg::RING);
  float *scales = reinterpret_cast<float *>(smem + Cfg::RING + Cfg::SUMS);
  uint64_t *bars = reinterpret_cast<uint64_t *>(scales + Cfg::SCALES);
  volatile int *abort_flag = reinterpret_cast<volatile int *>(bars + Cfg::WARPS * Cfg::STAGES);
  int *first_unit = reinterpret_cast<int *>(bars + Cfg::WARPS * Cfg::STAGES + 1);
  int *row0 = first_unit + a.groups + 1, *scan = row0 + a.groups + 1;
  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
  const bool one = elect_one();
  const int g = lane >> 2, t4 = lane & 3;
  const int wrow = ((g & 1) << 2) | (g & 2) | (g >> 2);   // the weight row of MMA row g (shared-memory banks)
  const uint32_t ring = tc::smem_u32(smem) + warp * (Cfg::STAGES * FEW_ITEM);
  const uint32_t bar = tc::smem_u32(bars) + warp * (Cfg::STAGES * 8);
  const int slices = (a.K + FEW_SLICE - 1) / FEW_SLICE, groups = (a.K + (1 << a.group_log2) - 1) >> a.group_log2;

  if (lane == 0) {
    for (int i = 0; i < Cfg::STAGES; ++i) tc::mbar_init(bar + 8 * i, 1);
    tc::fence_mbar_init();
  }
  if (tid == 0) {
    *abort_flag = 0;
    tc::prefetch_tmap(&weights);
  }
  pdl_trigger();
  int units = (a.M + TOKENS - 1) / TOKENS;
  if (!a.offsets) {
    // this block's rows are known: as much of them as may matter starts its way into L2
    // (with one unit; more units' rows are the same ones again)
    const uint32_t share = a.N / gridDim.x, over = a.N % gridDim.x, rows = share + (blockIdx.x < over ? 1 : 0);
    const uint8_t *w = a.w + (int64_t)(blockIdx.x * share + min(blockIdx.x, over)) * a.w_rs;
    const uint32_t bytes = min((uint32_t)(a.K + 1) / 2, (96u << 10) / max(1u, rows)) & ~15u;
    if (bytes && units == 1)
      for (uint32_t i = tid; i < rows; i += Cfg::THREADS) prefetch_l2_bulk(w + i * a.w_rs, bytes);
    pdl_wait();
    __syncthreads();
  } else {
    pdl_wait();
    units = unit_table(a, TOKENS, first_unit, row0, scan);
  }
  // this block's share of the units' rows (units * N stays below 2^32: checked by the host)
  const uint32_t total = (uint32_t)units * (uint32_t)a.N, share = total / gridDim.x, over = total % gridDim.x;
  uint32_t at = blockIdx.x * share + min(blockIdx.x, over);
  const uint32_t end = at + share + (blockIdx.x < over ? 1 : 0);
  int st = 0;            // the ring's next stage and its phase: the same for copies and reads
  uint32_t phase = 0;

  while (at < end) {
    // up to TILES row tiles of one unit
    const int u = (int)(at / (uint32_t)a.N), n0 = (int)(at - (uint32_t)u * (uint32_t)a.N);
    const int rows = (int)min(min(end - at, (uint32_t)(a.N - n0)), (uint32_t)(16 * Cfg::TILES));
    int e = 0, m0 = u * TOKENS, m1 = a.M;
    if (a.offsets) {
      e = group_of_unit(first_unit, a.groups, u);
      m0 = row0[e] + (u - first_unit[e]) * TOKENS;
      m1 = row0[e + 1];
    }
    m1 = min(m1, m0 + TOKENS);
    const int tiles = (rows + 15) / 16, we = a.w_e == 0 ? 0 : e;

    // the slices whose scales fit, at a time: with 7 row tiles K up to 17408 in groups of 128 (8448 with
    // zero points) or 4352 in groups of 32 (2048), with 4 tiles up to 30464 (15104) or 7424 (3584)
    float *own = sums + warp * (Cfg::TILES * NT * 128) + lane * 4;
    const int per_slice = max(1, FEW_SLICE >> a.group_log2);
    const int fit = max(1, (Cfg::SCALES / WORDS / (tiles * 16) - 1) / per_slice);
    for (int s0 = 0; s0 < slices; s0 += fit) {
      const int s1 = min(slices, s0 + fit), items = (s1 - s0) * tiles;
      const int i0 = items * warp / Cfg::WARPS, i1 = items * (warp + 1) / Cfg::WARPS;
      const int q_first = i0 / tiles, first = s0 + q_first, t_first = i0 - q_first * tiles;
      const int last = i0 < i1 ? s0 + (i1 - 1) / tiles : -1;
      int fs = first, ft = t_first, fetched = i0;   // the next item to fetch
      auto fetch = [&](int stage) {   // (by one lane)
        if (fetched >= i1) return;
        tc::mbar_arrive_expect_tx(bar + 8 * stage, FEW_ITEM);
        tc::tma_load_3d(ring + stage * FEW_ITEM, &weights, bar + 8 * stage, fs * (FEW_SLICE / 2), n0 + ft * 16, we);
        ++fetched;
        if (++ft == tiles) { ft = 0; ++fs; }
      };
      // a slice's tokens
      uint4 raw[NT][8];
      auto fetch_tokens = [&](int s) {
        const int k0 = s * FEW_SLICE + t4 * (8 * LW);
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const int m = m0 + n * 8 + g;
          const T *row = static_cast<const T *>(a.x) + (int64_t)m * a.x_rs + k0;
          const bool on = m < m1;
          if ((s + 1) * FEW_SLICE <= a.K) {
#pragma unroll
            for (int v = 0; v < 8; ++v) {
              raw[n][v] = make_uint4(0, 0, 0, 0);
              if (on) raw[n][v] = *reinterpret_cast<const uint4 *>(row + (v / LW) * SUB + (v % LW) * 8);
            }
          } else {   // (rows hold whole 16 bytes: the host has copied others)
#pragma unroll
            for (int v = 0; v < 8; ++v) {
              const int k = (v / LW) * SUB + (v % LW) * 8, left = a.K - k0 - k;
              Vec<T> w;
              w.zero();
              if (on && left > 0) w.u.q = *reinterpret_cast<const uint4 *>(row + k);
              keep_first(w, max(left, 0));
              raw[n][v] = w.u.q;
            }
          }
        }
      };
      if (one) {
        int stage = st;
#pragma unroll 1
        for (int i = 0; i < Cfg::STAGES; ++i) {
          fetch(stage);
          stage = stage + 1 == Cfg::STAGES ? 0 : stage + 1;
        }
      }
      if (i0 < i1) fetch_tokens(first);
      if (s0 == 0)
        for (int i = 0; i < tiles * NT; ++i) *reinterpret_cast<float4 *>(own + i * 128) = make_float4(0.f, 0.f, 0.f, 0.f);
      // scales of the rows, fp32; an odd pitch, so that eight rows meet eight banks;
      // and zeros for groups past the end, whose sums are zeros
      // (A row a warp, and all of its rows' loads on their way at a time or, where the block has few
      // rows, spans of two: one after another they were 4 of 19 us.)
      const int q0 = (s0 * FEW_SLICE) >> a.group_log2, qn = (s1 - s0) * per_slice, pitch = qn | 1;
      constexpr int BATCH = (16 * Cfg::TILES + Cfg::WARPS - 1) / Cfg::WARPS;
      const bool narrow = rows <= 2 * Cfg::WARPS;
      const int64_t i_s = e * a.s_e + (int64_t)(n0 + warp) * a.s_rs + q0 + lane;
      const int64_t i_z = e * a.z_e + (int64_t)(n0 + warp) * a.z_rs + q0 + lane;
      const int64_t step_s = Cfg::WARPS * a.s_rs, step_z = Cfg::WARPS * a.z_rs;
      for (int qb = 0; qb < qn; qb += narrow ? 32 * (BATCH / 2) : 32) {
        uint32_t v[BATCH];
        uint8_t z[BATCH];
#pragma unroll
        for (int j = 0; j < BATCH; ++j) {
          const int row = narrow ? j & 1 : j, q = qb + (narrow ? (j >> 1) * 32 : 0);
          const bool load = warp + row * Cfg::WARPS < rows && q + lane < qn && q0 + q + lane < groups;
          v[j] = load ? scale_bits<T>(a, i_s + row * step_s + q) : 0u;
          if constexpr (ZERO) z[j] = load ? a.zero[i_z + row * step_z + q] : 0;
        }
#pragma unroll
        for (int j = 0; j < BATCH; ++j) {
          const int row = narrow ? j & 1 : j, q = qb + (narrow ? (j >> 1) * 32 : 0) + lane, r = warp + row * Cfg::WARPS;
          if (r >= rows || q >= qn) continue;
          const float f = scale_of<T>(a, v[j]);
          if constexpr (ZERO) reinterpret_cast<float2 *>(scales)[r * pitch + q] = make_float2(f, (float)z[j]);
          else scales[r * pitch + q] = f;
        }
      }
      __syncthreads();

      uint32_t x[NT][8][4];
      int s = first, t = t_first, held = -1, i = i0;
      for (; i < i1; ++i) {
        if (s != held) {
          held = s;
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int v = 0; v < 8; ++v) token_pairs(raw[n][v], x[n][v]);
          if (s < last) fetch_tokens(s + 1);
        }
        if (!__all_sync(0xffffffffu, tc::mbar_wait(bar + 8 * st, phase, abort_flag, timeout_ns))) break;
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
                           : "=r"(q[h][4 * j]), "=r"(q[h][4 * j + 1]), "=r"(q[h][4 * j + 2]), "=r"(q[h][4 * j + 3]) : "r"(p) : "memory");
            else if constexpr (LW == 2)
              asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(q[h][2 * j]), "=r"(q[h][2 * j + 1]) : "r"(p) : "memory");
            else
              asm volatile("ld.shared.u32 %0, [%1];" : "=r"(q[h][j]) : "r"(p) : "memory");
          }
        }
        // every lane's loads are done before the copy over them is issued: a warp barrier alone lets
        // them complete behind it, and the next item's rows were read (1111 rows by 256 experts)
        tc::fence_proxy_async_smem();
        __syncwarp();
        if (one) fetch(st);
        if (++st == Cfg::STAGES) { st = 0; phase ^= 1u; }

        // (rows past the end have any numbers for scales: their sums are not stored)
        const float *sc = scales + WORDS * ((t * 16 + wrow) * pitch + (((s - s0) * FEW_SLICE) >> a.group_log2));
        float acc[NT][4];
#pragma unroll
        for (int n = 0; n < NT; ++n) acc[n][0] = acc[n][1] = acc[n][2] = acc[n][3] = 0.f;
#pragma unroll
        for (int j = 0; j < SUBS; ++j) {
          // groups of 256 columns are two sums of 128
          const int c = LW == 4 ? (a.group_log2 == 8 ? 0 : j) : j;
          float sv0, sv1, z0 = 8.f, z1 = 8.f;
          if constexpr (ZERO) {
            const float2 v0 = *reinterpret_cast<const float2 *>(sc + 2 * c), v1 = *reinterpret_cast<const float2 *>(sc + 2 * (8 * pitch + c));
            sv0 = v0.x; z0 = v0.y;
            sv1 = v1.x; z1 = v1.y;
          } else {
            sv0 = sc[c];
            sv1 = sc[8 * pitch + c];
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
            acc[n][0] = fmaf(d[n][0], sv0, acc[n][0]);
            acc[n][1] = fmaf(d[n][1], sv0, acc[n][1]);
            acc[n][2] = fmaf(d[n][2], sv1, acc[n][2]);
            acc[n][3] = fmaf(d[n][3], sv1, acc[n][3]);
          }
        }
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          float4 *o = reinterpret_cast<float4 *>(own + (t * NT + n) * 128);
          const float4 v = *o;
          *o = make_float4(v.x + acc[n][0], v.y + acc[n][1], v.z + acc[n][2], v.w + acc[n][3]);
        }
        if (++t == tiles) { t = 0; ++s; }
      }
      if (i < i1 && one) {
        // given up: the copies on their way land before the block can leave
        volatile int no_abort = 0;
        for (; i < fetched; ++i) {
          tc::mbar_wait(bar + 8 * st, phase, &no_abort, timeout_ns);
          if (++st == Cfg::STAGES) { st = 0; phase ^= 1u; }
        }
      }
      if (__syncthreads_or(*abort_flag)) return;
    }
    if (slices == 0) {
      for (int i = 0; i < tiles * NT; ++i) *reinterpret_cast<float4 *>(own + i * 128) = make_float4(0.f, 0.f, 0.f, 0.f);
      __syncthreads();
    }
    // four results of a tile: rows r and r + 8, tokens c and c + 1
    for (int i = tid; i < tiles * NT * 32; i += Cfg::THREADS) {
      const int l = i & 31, tn = i >> 5, tile = tn / NT, n = tn - tile * NT;
      float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int k = 0; k < Cfg::WARPS; ++k) {
        const float4 v = *reinterpret_cast<const float4 *>(sums + k * (Cfg::TILES * NT * 128) + tn * 128 + l * 4);
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
  if (a.offsets) zero_rest<T>(a, row0[a.groups], tid, Cfg::THREADS);
}

}  // namespace i4
}  // namespace mb
