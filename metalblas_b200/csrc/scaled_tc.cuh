// int8 products with a scale for each row of A ("token") and each column of B
// ("channel"), one B per group of rows, on the int8 tensor cores:
//
//   C[m, n] = (sum_k A[m, k] B_e[k, n]) scale_a[m] scale_b[e, n] + bias[n]
//
// for rows m of group e, offsets[e] <= m < offsets[e + 1]; rows at or past
// offsets[groups] are set to zero.  The sum is exact in 32-bit integers
// (K <= 131071); it is converted to fp32 once, multiplied by scale_a, then by
// scale_b, and bias is added: four fp32 roundings at most and one to the output
// type, the same for every tile and split, so a row's result does not depend on
// the rows beside it.
//
// Structure (the warp roles, the TMA -> 128B-swizzled ring -> tcgen05.mma ->
// TMEM pipeline and the bounded waits are tc_gemm.cuh's):
//   warp 0      TMA producer; warp 1 the MMA issuer (kind::i8, s32 in TMEM);
//   warps 2..9  epilogue, two warps per TMEM lane quarter.
// Persistent over units (group, row tile, channel tile).  The host knows the
// rows of a group only when there is one; otherwise every CTA reads the device
// offsets at its start and scans them into a table of unit counts in shared
// memory, and each role finds its unit there by bisection.  Empty groups have
// no unit.  A tile loads whole boxes of A rows, those of the next group
// included (integers: a stray row costs nothing), and stores only its own rows.
//
// SWAP = false: UMMA rows are tokens (128, or 256 on a CTA pair), columns are
//   channels: the compute-bound form.  A warp stages 32 rows x 32 columns in
//   shared memory and stores them as one TMA box; rows that end with a group
//   inside C (a box could only clip at the tensor's end) go out by 16-byte stores.
// SWAP = true: UMMA rows are 128 channels, columns 16..128 tokens: with few
//   rows per group the product is a stream of weights, and this form loads the
//   fewest other bytes per weight byte.  Lanes hold channels; the staged rows
//   are tokens all the same.
//
// split > 1 (few units): the CTAs of a cluster share one unit, each a range of
// K.  Eight epilogue warps hold eight pieces of the tile; piece i is finished
// by cluster rank i * split / 8, and the other ranks send it their s32 partial
// sums through distributed shared memory.
//
// What bounds it, measured on B200 by graph replay (twice the bf16 GEMM rate 1650
// TFLOP/s is taken as the int8 rate, 6.54 TB/s is a copy's):
//   8192^3 bf16 out                333 us, 3300 TOPS: the tensor pipe;
//   4096^3                         49.6 us, 2770 TOPS: operands into shared memory,
//                                  and 256 tiles over 74 pairs;
//   16384 rows by 8 experts of 4096 x 14336   662 us, 2910 TOPS: the same, and
//                                  tiles that end with their group;
//   8192 x 512 x 8192              49 us, 2.9 TB/s: latency of the epilogue, whose eight
//                                  warps an SM wait for one TMEM load, conversion and
//                                  store after another (issue slots 36 % in use, tensor
//                                  pipe 30 %, L2 29 %);
//   16 rows by 7 experts of 4096 x 14336      69.5 us, 5.9 TB/s: the weights' bytes;
//   16 x 4096 x 14336              14.2 us, 4.2 TB/s: 112 tiles keep 112 SMs busy;
//   17 to 1000 rows, one wave of tiles or less: the start, one tile's K loop and its
//                                  epilogue, one after another (1024 x 4096 x 2048 14.0
//                                  us: tensor pipe 22 %, DRAM 9 %, issue slots 13 %).
// The tile is chosen by sg_cost (mb_ops.cu), a model of such times; TROWS, TCOLS
// and split change no result.
#pragma once
#include "pack.cuh"
#include "quantize.cuh"
#include "tc_gemm.cuh"

namespace mb {
namespace sg {

using namespace mb::tc;

constexpr int kMaxGroups = 1024;
constexpr int MAX_STAGES = 12;
constexpr int TABLE_BYTES = 2 * (kMaxGroups + 1) * 4 + 56;
constexpr int BAR_BYTES = 512;

struct SgParams {
  CUtensorMap tmA, tmB;    // UMMA-A and UMMA-B operands, {inner, outer, group}
  CUtensorMap tmC;         // C, boxes of 32 x 32, for c_tma
  int M, N;                // tokens, channels
  int groups;
  const int *offsets;      // null: one group of all M rows
  int a_mn, b_mn;          // operand is MN-major in global memory
  int one_b;               // every group has the same B
  int K, kb_total, stages, split;
  const int8_t *w;         // SWAP, one group, K contiguous: the weights and their pitch
  int64_t w_ld;
  int tiles_c;             // channel tiles
  void *C;
  int64_t c_rs, c_cs;
  int c_tma;               // C has a tensor map
  int c_vec;               // c_cs == 1 and rows on 16-byte boundaries
  const float *scale_a, *scale_b;
  int64_t sa_s, sb_s, sb_g;
  const void *bias;        // per channel, or null
  int64_t bias_s;
  int bias_f32;
  unsigned long long timeout_ns;
};

template <int BN, int PAIR, bool SWAP, class TO>
struct SgCfg {
  using B = tc::Cfg<BN, 1, PAIR>;
  static_assert(B::NMMA == 1, "one MMA per K-step");
  static constexpr int TROWS = SWAP ? BN : BM * PAIR;   // token rows per tile
  static constexpr int TCOLS = SWAP ? BM : BN;          // channels per tile
  static constexpr int STAGE_BYTES = B::A_BYTES + B::B_BYTES;
  static constexpr int RB = 32 * (int)sizeof(TO);       // bytes of a staged row
  static constexpr int STAGING_WARP = (SWAP && BN < 64 ? BN / 2 : 32) * RB;  // rows a warp stores at a time
  static constexpr int VEC_WARP = 32 * 8;               // a chunk's column scales and biases
  static constexpr bool CAN_SPLIT = PAIR == 1 && BN <= 128;
  static constexpr int PIECE_BYTES = 64 * BN;   // 32 lanes x BN / 2 columns x 4 bytes
  static __host__ __device__ constexpr int red_bytes(int split) { return CAN_SPLIT ? (split - 1) * (8 / split) * PIECE_BYTES : 0; }
  static constexpr int fixed_bytes(int split) {
    return 1024 + NUM_EPI_WARPS * (STAGING_WARP + VEC_WARP) + red_bytes(split) + BAR_BYTES + TABLE_BYTES;
  }
  static constexpr int stages(int split) {
    const int n = (SMEM_LIMIT - fixed_bytes(split)) / STAGE_BYTES;
    return n > MAX_STAGES ? MAX_STAGES : n;
  }
  static constexpr int smem_bytes(int split) { return fixed_bytes(split) + stages(split) * STAGE_BYTES; }
  static_assert(stages(CAN_SPLIT ? 8 : 1) >= 3, "pipeline");
};

struct Tile {
  int e, r0, rend, c0;  // group, first token row, end of the group's rows, first channel
};

// Unit u of the table: groups in order; within a group channel tiles outside,
// up to 16 row tiles inside (concurrent CTAs share weight tiles in L2, and with
// many row tiles A panels too).
template <int TROWS, int TCOLS>
__device__ __forceinline__ Tile unit_tile(const int *first_unit, const int *row0, int groups, int tiles_c, int u) {
  int lo = 0, hi = groups;  // first_unit[lo] <= u < first_unit[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (first_unit[mid] <= u) lo = mid;
    else hi = mid;
  }
  Tile t;
  t.e = lo;
  const int v = u - first_unit[lo];
  const int tiles_r = (row0[lo + 1] - row0[lo] + TROWS - 1) / TROWS;
  const int per = 16 * tiles_c, g = v / per, w = v - g * per;
  const int gsz = min(tiles_r - g * 16, 16);
  t.r0 = row0[lo] + (g * 16 + w % gsz) * TROWS;
  t.rend = row0[lo + 1];
  t.c0 = (w / gsz) * TCOLS;
  return t;
}

template <class TO> __device__ __forceinline__ float bias_at(const SgParams &p, int64_t n) {
  if (p.bias_f32) return static_cast<const float *>(p.bias)[n * p.bias_s];
  return Elem<TO>::load(static_cast<const TO *>(p.bias)[n * p.bias_s], false);
}

// The value of a sum.  The roundings are spelled out: contracted to a fused
// multiply-add in one kernel and not in another, they would differ in the last bit.
__device__ __forceinline__ float scaled_sum(int sum, float scale_a, float scale_b) {
  return __fmul_rn(__fmul_rn(__int2float_rn(sum), scale_a), scale_b);
}

// Four sums of one row, two to an instruction: the same roundings.
__device__ __forceinline__ void scaled_sums(const int *sum, float scale_a, const float4 &scale_b, float *v) {
  const float2 sa = make_float2(scale_a, scale_a);
#pragma unroll
  for (int i = 0; i < 4; i += 2) {
    const float2 f = make_float2(__int2float_rn(sum[i]), __int2float_rn(sum[i + 1]));
    const float2 o = mul2(mul2(f, sa), i ? make_float2(scale_b.z, scale_b.w) : make_float2(scale_b.x, scale_b.y));
    v[i] = o.x;
    v[i + 1] = o.y;
  }
}

// Moves the words x[0 .. W-1] up by `bytes` (0 to 15), with the last bytes of `before` in front.
template <int W>
__device__ __forceinline__ void shift_up(uint32_t *x, std::integral_constant<int, W>, const uint4 &before, uint32_t bytes) {
  const uint32_t b[4] = {before.x, before.y, before.z, before.w};
  const bool two = bytes & 8, one = bytes & 4;
  uint32_t y[W + 2], z[W + 1];
#pragma unroll
  for (int k = -2; k < W; ++k) y[k + 2] = two ? (k < 2 ? b[(k + 2) & 3] : x[k < 2 ? 0 : k - 2]) : (k < 0 ? b[(k + 4) & 3] : x[k < 0 ? 0 : k]);
#pragma unroll
  for (int k = 0; k <= W; ++k) z[k] = one ? y[k] : y[k + 1];
#pragma unroll
  for (int k = 0; k < W; ++k) x[k] = __funnelshift_l(z[k], z[k + 1], (bytes & 3) * 8);
}
// Bytes past .. 15 (store_from) and 0 .. past-1 (store_up_to) of a 16-byte chunk, past a
// multiple of TO's size and not 0, as 8, 4 and 2 bytes.
template <class TO> __device__ __forceinline__ void store_from(char *chunk, const uint32_t *w, uint32_t past) {
  if (past <= 8) *reinterpret_cast<uint2 *>(chunk + 8) = make_uint2(w[2], w[3]);
  const uint32_t up4 = (past + 3) & ~3u;  // the first whole word
  if (up4 & 4) *reinterpret_cast<uint32_t *>(chunk + up4) = up4 & 8 ? w[3] : w[1];
  if constexpr (sizeof(TO) == 2) {
    const uint32_t i = past >> 2, word = i & 2 ? (i & 1 ? w[3] : w[2]) : (i & 1 ? w[1] : w[0]);
    if (past & 2) *reinterpret_cast<uint16_t *>(chunk + past) = (uint16_t)(word >> 16);
  }
}
template <class TO> __device__ __forceinline__ void store_up_to(char *chunk, const uint32_t *w, uint32_t past) {
  if (past & 8) *reinterpret_cast<uint2 *>(chunk) = make_uint2(w[0], w[1]);
  if (past & 4) *reinterpret_cast<uint32_t *>(chunk + (past & 8)) = past & 8 ? w[2] : w[0];
  if constexpr (sizeof(TO) == 2) {
    const uint32_t i = past >> 2, word = i & 2 ? (i & 1 ? w[3] : w[2]) : (i & 1 ? w[1] : w[0]);
    if (past & 2) *reinterpret_cast<uint16_t *>(chunk + (past & 12)) = (uint16_t)word;
  }
}

// 4 consecutive results as the words of a staged row.
template <class TO> __device__ __forceinline__ void pack4(const float *v, uint32_t *w) {
  if constexpr (sizeof(TO) == 4) {
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = __float_as_uint(v[i]);
  } else {
    TO t[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) t[i] = Elem<TO>::store(v[i]);
    w[0] = reinterpret_cast<uint32_t *>(t)[0];
    w[1] = reinterpret_cast<uint32_t *>(t)[1];
  }
}

// RUNS: rows of C are contiguous but off 16 bytes (a kernel of its own: the shifts
// cost the others 10% where the epilogue binds, 5551 x 512 x 9312 39.8 us).
template <int BN, int PAIR, bool SWAP, bool RUNS, class TO>
__global__ void __launch_bounds__(NUM_THREADS, 1) scaled_gemm_kernel(const __grid_constant__ SgParams p) {
  using C_ = SgCfg<BN, PAIR, SWAP, TO>;
  using B_ = typename C_::B;
  constexpr int BK = 128;
  constexpr uint32_t A_BYTES = B_::A_BYTES, STAGE_BYTES = C_::STAGE_BYTES;
  const int stages = p.stages, split = C_::CAN_SPLIT ? p.split : 1;

  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t *ring = smem;
  uint8_t *staging = ring + stages * STAGE_BYTES;
  uint8_t *vecs = staging + NUM_EPI_WARPS * C_::STAGING_WARP;
  uint8_t *red = vecs + NUM_EPI_WARPS * C_::VEC_WARP;
  uint64_t *bars = reinterpret_cast<uint64_t *>(red + C_::red_bytes(split));
  int *first_unit = reinterpret_cast<int *>(reinterpret_cast<uint8_t *>(bars) + BAR_BYTES);
  int *row0 = first_unit + p.groups + 1;
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(bars + 2 * MAX_STAGES + 7);
  volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);
  int *scan = reinterpret_cast<int *>(tmem_slot + 2);  // a word per warp

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t ring_u32 = smem_u32(ring), bar_u32 = smem_u32(bars);
  auto full_bar = [&](int s) { return bar_u32 + 8u * s; };
  auto empty_bar = [&](int s) { return bar_u32 + 8u * (MAX_STAGES + s); };
  auto tfull_bar = [&](int a) { return bar_u32 + 8u * (2 * MAX_STAGES + a); };
  auto tempty_bar = [&](int a) { return bar_u32 + 8u * (2 * MAX_STAGES + 2 + a); };
  const uint32_t drain_bar = bar_u32 + 8u * (2 * MAX_STAGES + 4);
  const uint32_t red_full = bar_u32 + 8u * (2 * MAX_STAGES + 5);   // partial sums have come from every other rank
  const uint32_t red_free = bar_u32 + 8u * (2 * MAX_STAGES + 6);   // every rank has read what this CTA sent
  const int csize = PAIR == 2 ? 2 : split;
  const uint32_t rank = csize > 1 ? cluster_rank() : 0u;
  const int cid = blockIdx.x / csize, ncl = gridDim.x / csize;
  auto leader_full = [&](int s) { return mapa_shared(full_bar(s), 0); };
  auto wait_x = [&](uint32_t bar, uint32_t parity) {
    if constexpr (PAIR == 2) return mbar_wait_cluster(bar, parity, abort_flag, p.timeout_ns);
    else return mbar_wait(bar, parity, abort_flag, p.timeout_ns);
  };

  pdl_trigger();
  if (threadIdx.x == 0) {
    for (int s = 0; s < stages; ++s) {
      mbar_init(full_bar(s), 1);
      mbar_init(empty_bar(s), 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(tfull_bar(a), 1);
      mbar_init(tempty_bar(a), NUM_EPI_WARPS * PAIR);
    }
    mbar_init(drain_bar, 1);
    if (split > 1) {
      // lane 0 of each sending warp; lane 0 of each finishing warp
      mbar_init(red_full, (split - 1) * (8 / split));
      mbar_init(red_free, (split - 1) * (8 / split));
    }
    *abort_flag = 0;
    fence_mbar_init();
    prefetch_tmap(&p.tmA);
    prefetch_tmap(&p.tmB);
  }
  if (warp == 1) {
    tmem_alloc_g<PAIR>(smem_u32(tmem_slot), B_::TMEM_COLS);
    tmem_relinquish_g<PAIR>();
  }
  tc_fence_before();
  __syncthreads();
  if (csize > 1) cluster_sync_all();  // every CTA's barriers are initialised before any remote arrival
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  // One group: this CTA's first unit is known, and its weights' way into L2 (as
  // much of them as the ring holds) may begin while the previous kernel ends.
  if (SWAP && p.w && threadIdx.x >= 64 && threadIdx.x < 64 + BM) {
    const int64_t n = (int64_t)(cid % p.tiles_c) * C_::TCOLS + (threadIdx.x - 64);
    const int k0 = split > 1 ? (int)((int64_t)rank * p.kb_total / split) * BK : 0;
    const int bytes = (min(p.K, k0 + stages * BK) - k0) & ~15;
    if (n < p.N && bytes > 0) prefetch_l2_bulk(p.w + n * p.w_ld + k0, (uint32_t)bytes);
  }
  pdl_wait();
  // The unit table: row0[e] and first_unit[e] for e <= groups.
  const int G = p.groups;
  if (!p.offsets) {
    if (threadIdx.x == 0) {
      row0[0] = 0;
      row0[1] = p.M;
      first_unit[0] = 0;
      first_unit[1] = (p.M + C_::TROWS - 1) / C_::TROWS * p.tiles_c;
    }
  } else {
    for (int e = threadIdx.x; e <= G; e += NUM_THREADS) row0[e] = e ? min(max(p.offsets[e], 0), p.M) : 0;
    __syncthreads();
    // Offsets that are not ascending name no groups: every row comes out as zeros
    // (and no count below can leave the range the host has checked).
    int wrong = 0;
    for (int e = threadIdx.x; e < G; e += NUM_THREADS) wrong |= row0[e + 1] < row0[e];
    if (__syncthreads_or(wrong)) {
      for (int e = threadIdx.x; e <= G; e += NUM_THREADS) row0[e] = 0;
      __syncthreads();
    }
    // each thread sums `per` consecutive groups, then a scan over threads
    const int per = (G + NUM_THREADS - 1) / NUM_THREADS;
    const int e0 = min(G, (int)threadIdx.x * per), e1 = min(G, e0 + per);
    auto units_of = [&](int e) { return (row0[e + 1] - row0[e] + C_::TROWS - 1) / C_::TROWS * p.tiles_c; };
    int sum = 0;
    for (int e = e0; e < e1; ++e) sum += units_of(e);
    int upto = sum;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int o = __shfl_up_sync(0xffffffffu, upto, d);
      if (lane >= d) upto += o;
    }
    if (lane == 31) scan[warp] = upto;
    __syncthreads();
    int at = upto - sum;
    for (int w = 0; w < warp; ++w) at += scan[w];
    for (int e = e0; e < e1; ++e) {
      first_unit[e] = at;
      at += units_of(e);
    }
    if (threadIdx.x == NUM_THREADS - 1) first_unit[G] = at;
  }
  __syncthreads();
  const int num_units = first_unit[G];

  if (warp == 0) {
    // ------------------------------------------------------------ producer
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      int issued_stage = -1;
      uint32_t issued_phase = 0;
      const int kb0 = split > 1 ? (int)((int64_t)rank * p.kb_total / split) : 0;
      const int kb1 = split > 1 ? (int)((int64_t)(rank + 1) * p.kb_total / split) : p.kb_total;
      for (int u = cid; u < num_units; u += ncl) {
        const Tile t = unit_tile<C_::TROWS, C_::TCOLS>(first_unit, row0, G, p.tiles_c, u);
        const int prank = PAIR == 2 ? (int)rank : 0;
        const int a0 = (SWAP ? t.c0 : t.r0) + prank * BM, b0 = SWAP ? t.r0 : t.c0;
        const int wg = p.one_b ? 0 : t.e;
        const int ag = SWAP ? wg : 0, bg = SWAP ? 0 : wg;
        for (int kb = kb0; kb < kb1; ++kb) {
          if (!wait_x(empty_bar(stage), phase ^ 1u)) goto producer_done;
          if (prank == 0) mbar_arrive_expect_tx(full_bar(stage), STAGE_BYTES * PAIR);
          const uint32_t sa = ring_u32 + stage * STAGE_BYTES, sb = sa + A_BYTES;
          auto load = [&](uint32_t dst, const CUtensorMap *map, int x, int y, int z) {
            if constexpr (PAIR == 2) tma_load_3d_pair(dst, map, leader_full(stage), x, y, z);
            else tma_load_3d(dst, map, full_bar(stage), x, y, z);
          };
          if (SWAP && p.a_mn) load(sa, &p.tmA, a0, kb * BK, ag);
          else load(sa, &p.tmA, kb * BK, a0, ag);
          // this CTA's share of the MMA's columns (see tc_gemm.cuh)
          constexpr int SH = B_::UMMA_N / PAIR;
          const int col = b0 + prank * SH;
          if (!SWAP && p.b_mn) {
#pragma unroll
            for (int j = 0; j < SH / 128; ++j) load(sb + j * (BK * 128), &p.tmB, col + j * 128, kb * BK, bg);
          } else {
            load(sb, &p.tmB, kb * BK, col, bg);
          }
          issued_stage = stage;
          issued_phase = phase;
          if (++stage == stages) { stage = 0; phase ^= 1u; }
        }
      }
    producer_done:
      // the last copies must land before the CTA can exit
      if (issued_stage >= 0) {
        volatile int no_abort = 0;
        if (PAIR == 1 || rank == 0) mbar_wait(full_bar(issued_stage), issued_phase, &no_abort, p.timeout_ns);
        else mbar_wait_cluster(empty_bar(issued_stage), issued_phase, &no_abort, p.timeout_ns);
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer
    if ((PAIR == 1 || rank == 0) && lane == 0) {
      const uint32_t idesc = make_idesc<int8_t, B_::UMMA_N, BM * PAIR>(SWAP ? p.a_mn : 0, SWAP ? 0 : p.b_mn);
      const bool amn = SWAP && p.a_mn, bmn = !SWAP && p.b_mn;
      const uint32_t a_lbo = amn ? BK * 128 : 16, b_lbo = bmn ? BK * 128 : 16;
      const uint32_t a_kstep = amn ? B_::UMMA_K * 128 : 32, b_kstep = bmn ? B_::UMMA_K * 128 : 32;
      const int kb0 = split > 1 ? (int)((int64_t)rank * p.kb_total / split) : 0;
      const int kb1 = split > 1 ? (int)((int64_t)(rank + 1) * p.kb_total / split) : p.kb_total;
      int stage = 0;
      uint32_t phase = 0;
      int abuf = 0;
      uint32_t aphase = 0;
      bool issued_any = false, aborted = false;
      for (int u = cid; u < num_units && !aborted; u += ncl) {
        if (!wait_x(tempty_bar(abuf), aphase ^ 1u)) break;
        tc_fence_after();
        const uint32_t d_tmem = tmem_base + (uint32_t)(abuf * B_::ACC_COLS);
        for (int kb = kb0; kb < kb1; ++kb) {
          if (!wait_x(full_bar(stage), phase)) { aborted = true; break; }
          tc_fence_after();
          const uint32_t sa = ring_u32 + stage * STAGE_BYTES, sb = sa + A_BYTES;
#pragma unroll
          for (int ks = 0; ks < B_::KSTEPS; ++ks) {
            const uint64_t ad = sdesc(sa + ks * a_kstep, a_lbo, 1024), bd = sdesc(sb + ks * b_kstep, b_lbo, 1024);
            umma_g<1, PAIR>(d_tmem, ad, bd, idesc, (kb > kb0 || ks > 0) ? 1u : 0u);
          }
          issued_any = true;
          umma_commit_g<PAIR>(empty_bar(stage));
          if (++stage == stages) { stage = 0; phase ^= 1u; }
        }
        if (aborted) break;
        umma_commit_g<PAIR>(tfull_bar(abuf));
        if (++abuf == B_::NACC) { abuf = 0; aphase ^= 1u; }
      }
      if (*abort_flag && issued_any) {
        umma_commit_self<PAIR>(drain_bar);
        volatile int no_abort = 0;
        mbar_wait(drain_bar, 0, &no_abort, p.timeout_ns);
      }
    }
  } else {
    // ------------------------------------------------------------ epilogue
    const int ew = warp - 2, q = warp & 3, half = ew >> 2;
    const uint32_t stg = smem_u32(staging) + (uint32_t)(ew * C_::STAGING_WARP);
    float *vec = reinterpret_cast<float *>(vecs + ew * C_::VEC_WARP);  // [32] scales, [32] biases
    TO *C = static_cast<TO *>(p.C);
    constexpr int WCOLS = BN / 2;                    // columns of this warp
    constexpr int CH = WCOLS < 32 ? WCOLS : 32;      // columns per step
    auto release_tmem = [&](int a) {
      if constexpr (PAIR == 2) mbar_arrive_cluster(mapa_shared(tempty_bar(a), 0));
      else mbar_arrive(tempty_bar(a));
    };
    // whole warps go on or give up: a lane whose limit ran out takes the others along
    auto all = [](bool ok) { return __all_sync(0xffffffffu, ok) != 0; };
    // Rows of no group.
    if (p.offsets) {
      const int64_t z0 = row0[G], zr = p.M - z0;
      const int tid = blockIdx.x * (NUM_EPI_WARPS * 32) + ew * 32 + lane;
      const int step = gridDim.x * (NUM_EPI_WARPS * 32);
      if (p.c_vec) {
        constexpr int EPC = 16 / (int)sizeof(TO);
        const int64_t nv = (p.N + EPC - 1) / EPC;
        for (int64_t i = tid; i < zr * nv; i += step) {
          const int64_t r = i / nv, n = (i - r * nv) * EPC;
          TO *dst = C + (z0 + r) * p.c_rs + n;
          if (n + EPC <= p.N) *reinterpret_cast<uint4 *>(dst) = make_uint4(0, 0, 0, 0);
          else
            for (int j = 0; n + j < p.N; ++j) dst[j] = Elem<TO>::store(0.f);
        }
      } else {
        for (int64_t i = tid; i < zr * p.N; i += step) {
          const int64_t r = i / p.N, n = i - r * p.N;
          C[(z0 + r) * p.c_rs + n * p.c_cs] = Elem<TO>::store(0.f);
        }
      }
    }
    // With split ranks: the piece of the tile this warp holds, the rank that
    // finishes it, and where its sums go there.
    const int piece = q * 2 + half, per_rank = 8 / split;
    const int owner = piece / per_rank, me = (int)rank;
    const uint32_t red_u32 = smem_u32(red) + (uint32_t)(piece % per_rank) * C_::PIECE_BYTES + (uint32_t)lane * 16u;
    const uint32_t red_step = (uint32_t)(per_rank * C_::PIECE_BYTES);  // from one source rank to the next
    uint32_t rphase = 0;
    bool first = true;

    int abuf = 0;
    uint32_t aphase = 0;
    for (int u = cid; u < num_units; u += ncl) {
      const Tile t = unit_tile<C_::TROWS, C_::TCOLS>(first_unit, row0, G, p.tiles_c, u);
      // The scales are on their way while the accumulator fills: this lane's row (a
      // token, or a channel when swapped) and, a column per lane, the first columns.
      const int row = (PAIR == 2 ? (int)rank * BM : 0) + q * 32 + lane;   // UMMA row of this lane
      const int64_t m = t.r0 + row, n = t.c0 + row;
      const bool finish = split == 1 || owner == me;
      float rs = 0.f, rb = 0.f, cs_next = 0.f, cb_next = 0.f;
      auto load_cols = [&](int c) {
        const int64_t col = (SWAP ? t.r0 : t.c0) + half * WCOLS + c + lane;
        cs_next = cb_next = 0.f;
        if constexpr (SWAP) {
          if (lane < CH && col < t.rend) cs_next = p.scale_a[col * p.sa_s];
        } else {
          if (lane < CH && col < p.N) {
            cs_next = p.scale_b[t.e * p.sb_g + col * p.sb_s];
            if (p.bias) cb_next = bias_at<TO>(p, col);
          }
        }
      };
      if (finish) {
        if constexpr (SWAP) {
          if (n < p.N) {
            rs = p.scale_b[t.e * p.sb_g + n * p.sb_s];
            if (p.bias) rb = bias_at<TO>(p, n);
          }
        } else {
          if (m < t.rend) rs = p.scale_a[m * p.sa_s];
        }
        load_cols(0);
      }
      if (!all(wait_x(tfull_bar(abuf), aphase))) break;
      tc_fence_after();
      const uint32_t tbase = tmem_base + ((uint32_t)(q * 32) << 16) + (uint32_t)(abuf * B_::ACC_COLS + half * WCOLS);
      if (!finish) {
        // what this CTA sent for the last unit has been read
        if (!first && !all(mbar_wait_cluster(red_free, rphase ^ 1u, abort_flag, p.timeout_ns))) break;
        const uint32_t dst = mapa_shared(red_u32 + (uint32_t)(me - (me > owner ? 1 : 0)) * red_step, (uint32_t)owner);
#pragma unroll 1
        for (int c = 0; c < WCOLS; c += CH) {
          uint32_t r[32];
          tmem_ld<CH>(tbase + c, r);
          tmem_wait_ld();
#pragma unroll
          for (int j = 0; j < CH; j += 4)
            st_cluster_v4(dst + (uint32_t)((c + j) >> 2) * 512u, r[j], r[j + 1], r[j + 2], r[j + 3]);
        }
        tc_fence_before();
        __syncwarp();  // the lanes' stores come before lane 0's release
        if (lane == 0) {
          mbar_arrive_cluster(mapa_shared(red_full, (uint32_t)owner));
          release_tmem(abuf);
        }
      } else {
        if (split > 1 && !all(mbar_wait_cluster(red_full, rphase, abort_flag, p.timeout_ns))) break;
        static_assert(!(SWAP && RUNS), "lanes hold rows");
        uint4 rest = make_uint4(0, 0, 0, 0);  // RUNS: the row's last chunk as converted
#pragma unroll 1
        for (int c = 0; c < WCOLS; c += CH) {
          uint32_t r[32];
          tmem_ld<CH>(tbase + c, r);
          const float cs = cs_next, cb = cb_next;
          if (c + CH < WCOLS) load_cols(c + CH);
          __syncwarp();  // the last step's reads of vec and of the staging rows are done
          vec[lane] = cs;
          if constexpr (!SWAP) vec[32 + lane] = cb;
          __syncwarp();
          tmem_wait_ld();
          if (c + CH >= WCOLS) {  // the accumulator is read
            tc_fence_before();
            __syncwarp();
            if (lane == 0) release_tmem(abuf);
          }
          if (split > 1) {
#pragma unroll 1
            for (int s = 0; s < split - 1; ++s) {
#pragma unroll
              for (int j = 0; j < CH; j += 4) {
                const uint4 v = ld_shared_v4(red_u32 + s * red_step + (uint32_t)((c + j) >> 2) * 512u);
                r[j] += v.x; r[j + 1] += v.y; r[j + 2] += v.z; r[j + 3] += v.w;
              }
            }
          }
          constexpr int EPC = 16 / (int)sizeof(TO);   // elements per 16-byte chunk
          constexpr int NCH = C_::RB / 16;            // chunks per staged row
          auto chunk_addr = [&](int rr, int ch) {
            // Written by rows (a lane a row), rows 8 (16-bit) or 4 apart would share
            // banks; written by columns (swapped) they lie as they are.
            const int x = SWAP ? 0 : NCH == 4 ? (rr >> 1) & 3 : rr & 7;
            return stg + (uint32_t)(rr * C_::RB) + ((uint32_t)(ch ^ x) << 4);
          };
          if constexpr (SWAP) {
            TO *col = reinterpret_cast<TO *>(staging + ew * C_::STAGING_WARP) + lane;
#pragma unroll
            for (int j = 0; j < CH; j += 4) {
              const float4 s4 = *reinterpret_cast<const float4 *>(vec + j);
              const float sc[4] = {s4.x, s4.y, s4.z, s4.w};
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                float v = scaled_sum((int)r[j + i], sc[i], rs);
                if (p.bias) v = __fadd_rn(v, rb);
                col[(j + i) * 32] = Elem<TO>::store(v);
              }
            }
          } else {
            static_assert(CH == 32, "whole staged rows");
            uint32_t w[NCH][4];
            auto convert = [&](auto with_bias) {
#pragma unroll
              for (int j = 0; j < 32; j += 4) {
                const float4 s4 = *reinterpret_cast<const float4 *>(vec + j);
                float v[4];
                scaled_sums(reinterpret_cast<const int *>(r) + j, rs, s4, v);
                if constexpr (decltype(with_bias)::value) {
                  const float4 b4 = *reinterpret_cast<const float4 *>(vec + 32 + j);
                  v[0] = __fadd_rn(v[0], b4.x); v[1] = __fadd_rn(v[1], b4.y);
                  v[2] = __fadd_rn(v[2], b4.z); v[3] = __fadd_rn(v[3], b4.w);
                }
                pack4<TO>(v, &w[j / EPC][sizeof(TO) == 4 ? 0 : j % 8 / 2]);
              }
            };
            if (p.bias) convert(std::true_type());
            else convert(std::false_type());
            if (p.c_rs == 1 && p.c_cs != 1) {  // columns of C are contiguous: lanes hold rows
              const int64_t r = t.r0 + row, n0 = t.c0 + half * WCOLS + c;
#pragma unroll
              for (int j = 0; j < 32; ++j)
                if (r < t.rend && n0 + j < p.N) C[r + (n0 + j) * p.c_cs] = reinterpret_cast<const TO *>(w)[j];
              continue;
            }
            const int64_t nn = t.c0 + half * WCOLS + c;
            if constexpr (RUNS) if (nn + 32 <= p.N) {
              // A row that starts anywhere: its 32 elements move up to the 16-byte chunks of
              // C that hold them, with the last chunk's rest before them.  What is left
              // over at either end of the warp's columns goes out by itself.  (5551 x 512 x
              // 9315 bf16 53 us; an element a lane 85, with chunks cut out of the staged
              // rows 87; rows of 9312 40.)
              TO *own = C + m * p.c_rs + nn;
              const uint32_t past = (uint32_t)(reinterpret_cast<uintptr_t>(own) & 15);
              char *chunk = reinterpret_cast<char *>(own) - past;
              const uint4 end = make_uint4(w[NCH - 1][0], w[NCH - 1][1], w[NCH - 1][2], w[NCH - 1][3]);
              shift_up(&w[0][0], std::integral_constant<int, NCH * 4>(), rest, past);
              if (c == 0 && past && m < t.rend) store_from<TO>(chunk, w[0], past);
              if ((c + CH >= WCOLS || nn + 64 > p.N) && past && m < t.rend) {
                uint32_t tail[4] = {0, 0, 0, 0};
                shift_up(tail, std::integral_constant<int, 4>(), end, past);
                store_up_to<TO>(chunk + 32 * sizeof(TO), tail, past);
              }
              rest = end;
            }
            if (!RUNS && p.c_tma) {  // the last step's store has read the staging rows
              if (lane == 0) bulk_wait_read0();
              __syncwarp();
            }
#pragma unroll
            for (int ch = 0; ch < NCH; ++ch)
              asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(chunk_addr(lane, ch)), "r"(w[ch][0]),
                           "r"(w[ch][1]), "r"(w[ch][2]), "r"(w[ch][3])
                           : "memory");
            // 32 rows of the group (or up to the end of C, where the store clips)
            // go out as one box; the rows before another group's by hand, and so the
            // columns before an end off 16 bytes: along them the store clips whole
            // chunks alone, and wrote up to 14 bytes past a row of N = 33.
            const int64_t first_row = t.r0 + (PAIR == 2 ? (int)rank * BM : 0) + q * 32;
            if (!RUNS && p.c_tma && (first_row + 32 <= t.rend || t.rend == p.M) && (nn + 32 <= p.N || p.N % EPC == 0)) {
              fence_proxy_async_smem();
              __syncwarp();
              if (lane == 0 && first_row < t.rend && nn < p.N) {
                tma_store_3d(&p.tmC, stg, (int)nn, (int)first_row, 0);
                bulk_commit();
              }
              continue;
            }
          }
          __syncwarp();
          constexpr int ROWS = SWAP ? CH : 32, PASS = 32 / NCH;
          const int64_t mw = SWAP ? t.r0 + half * WCOLS + c : t.r0 + (PAIR == 2 ? (int)rank * BM : 0) + q * 32;
          const int64_t nw = SWAP ? t.c0 + q * 32 : t.c0 + half * WCOLS + c;
          const int live = (int)min((int64_t)ROWS, t.rend - mw);   // rows of the group among them
          if (!RUNS && p.c_vec && nw + 32 <= p.N) {
            // 16-byte chunks, whole rows by neighbouring lanes
            const int ch = lane % NCH, rr0 = lane / NCH;
#pragma unroll
            for (int i = 0; i < (ROWS + PASS - 1) / PASS; ++i) {
              const int rr = i * PASS + rr0;
              if (rr < live)
                *reinterpret_cast<uint4 *>(C + (mw + rr) * p.c_rs + nw + ch * EPC) = ld_shared_v4(chunk_addr(rr, ch));
            }
          } else if (RUNS && nw + 32 <= p.N) {
            // the staged chunks lie on 16 bytes of their rows; the first one of the
            // warp's columns has been stored by its lane where it is not whole
            const int ch = lane % NCH, rr0 = lane / NCH;
            const TO *dst = C + (mw + rr0) * p.c_rs + nw;
#pragma unroll
            for (int i = 0; i < (ROWS + PASS - 1) / PASS; ++i, dst += PASS * p.c_rs) {
              const int rr = i * PASS + rr0;
              const uintptr_t at = reinterpret_cast<uintptr_t>(dst);
              if (rr < live && (c | ch || at % 16 == 0))
                *reinterpret_cast<uint4 *>((at & ~uintptr_t(15)) + ch * 16) = ld_shared_v4(chunk_addr(rr, ch));
            }
          } else {
            // columns of C, the last ones of its rows, or any strides: an element a
            // lane, along whichever of rows and columns is contiguous
            const uint8_t *own = staging + ew * C_::STAGING_WARP;
            auto staged = [&](int rr, int col) {
              return *reinterpret_cast<const TO *>(own + (chunk_addr(rr, col / EPC) - stg) + (col % EPC) * sizeof(TO));
            };
            if (p.c_rs == 1 && p.c_cs != 1) {
#pragma unroll 4
              for (int col = 0; col < 32; ++col)
                if (lane < live && nw + col < p.N) C[mw + lane + (nw + col) * p.c_cs] = staged(lane, col);
            } else if (nw + lane < p.N) {
#pragma unroll 4
              for (int rr = 0; rr < live; ++rr) C[(mw + rr) * p.c_rs + (nw + lane) * p.c_cs] = staged(rr, lane);
            }
          }
        }
        if (split > 1) {
          __syncwarp();
          if (lane < split && lane != me) mbar_arrive_cluster(mapa_shared(red_free, (uint32_t)lane));
        }
      }
      rphase ^= 1u;
      first = false;
      if (++abuf == B_::NACC) { abuf = 0; aphase ^= 1u; }
    }
    if (!SWAP && lane == 0) bulk_wait0();  // this warp's stores have been made
    __syncwarp();
  }

  tc_fence_before();
  __syncthreads();
  if (csize > 1) cluster_sync_all();  // no CTA leaves while others still reach its shared memory
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_g<PAIR>(tmem_base, B_::TMEM_COLS);
  }
}

// Operands that TMA cannot read in place, copied to aligned rows: A's rows by the
// first `split` blocks, B's by the others, in one launch.  A lane takes 16 bytes of
// a row at a time and the lanes run on through rows; the bytes past a row's end go to its
// padding, which no tensor map covers.  Weights of groups without rows (offsets:
// of the groups; null: all have some) are left where they are: no unit reads them,
// and copying them all was most of a call with few rows (4 rows, 128 groups of 431 x
// 8192: 276 us, 26 now; 1024 x 4 rows, 32 groups of 4095 x 2048: 199, 190).
__global__ static void __launch_bounds__(256, 4) scaled_pack_kernel(const PackArgs pa, const PackArgs pb, int split,
                                                                 const int *offsets, int M) {
  __shared__ uint16_t used[1024];  // groups with rows
  __shared__ int count[8];
  pdl_trigger();
  pdl_wait();
  const bool is_a = (int)blockIdx.x < split;
  const PackArgs &a = is_a ? pa : pb;
  const int block = is_a ? blockIdx.x : blockIdx.x - split, blocks = is_a ? split : gridDim.x - split;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int batch = (int)a.batch;
  const bool some = !is_a && offsets;
  if (some) {
    const int groups = batch;
    batch = 0;
    for (int e0 = 0; e0 < groups; e0 += 256) {
      const int e = e0 + threadIdx.x;
      const bool has = e < groups && min(max(offsets[e + 1], 0), M) > (e ? min(max(offsets[e], 0), M) : 0);
      const unsigned mask = __ballot_sync(0xffffffffu, has);
      if (lane == 0) count[warp] = __popc(mask);
      __syncthreads();
      int at = batch + __popc(mask & ((1u << lane) - 1));
      for (int w = 0; w < 8; ++w) {
        at += w < warp ? count[w] : 0;
        batch += count[w];
      }
      if (has) used[at] = (uint16_t)e;
      __syncthreads();
    }
  }
  // vectors numbered through the rows; a thread's are `step` apart: dn batches, dr rows, dc vectors
  // (r + dr can pass 31 bits)
  const uint32_t vecs = (uint32_t)((a.cols + 15) / 16), rows = (uint32_t)a.rows;
  const uint32_t step = blocks * 256, at = block * 256 + threadIdx.x;
  const uint32_t dc = step % vecs, dr = step / vecs % rows, dn = step / vecs / rows;
  uint32_t c = at % vecs, r = at / vecs % rows;
  int n = (int)(at / vecs / rows);
  while (n < batch) {
    // four words on their way at a time; those without a byte of the row are not read
    uint4 lo[4], hi[4];
    uint32_t off[4];
    int8_t *dst[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const bool on = n < batch;
      const int64_t b = on ? (some ? used[n] : n) : 0;
      const int8_t *src = static_cast<const int8_t *>(a.src) + b * a.bs + (int64_t)r * a.rs + c * 16;
      off[i] = (uint32_t)(reinterpret_cast<uintptr_t>(src) & 15);
      lo[i] = load_once<true>(src - off[i], on);
      hi[i] = load_once<true>(src - off[i] + 16, on && off[i] && c * 16 + 16 - off[i] < (uint32_t)a.cols);
      dst[i] = on ? static_cast<int8_t *>(a.dst) + (b * (int64_t)rows + r) * a.ld + c * 16 : nullptr;
      c += dc;
      r += dr;
      n += (int)dn;
      if (c >= vecs) { c -= vecs; ++r; }
      if (r >= rows) { r -= rows; ++n; }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (dst[i]) *reinterpret_cast<uint4 *>(dst[i]) = cut16(lo[i], hi[i], off[i]);
  }
}

// K = 0: the sum is empty.  (Offsets that are not ascending name no groups, as
// in the other kernels.)
template <class TO>
__global__ void __launch_bounds__(256) scaled_empty_kernel(const SgParams p) {
  pdl_trigger();
  pdl_wait();
  int wrong = 0;
  if (p.offsets)
    for (int e = threadIdx.x + 1; e < p.groups; e += 256)
      wrong |= min(max(p.offsets[e + 1], 0), p.M) < min(max(p.offsets[e], 0), p.M);
  wrong = __syncthreads_or(wrong);
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < (int64_t)p.M * p.N; i += (int64_t)gridDim.x * 256) {
    const int64_t m = i / p.N, n = i - m * p.N;
    int e = 0;
    if (p.offsets) {
      if (wrong) e = p.groups;
      while (e < p.groups && m >= p.offsets[e + 1]) ++e;
    }
    float v = 0.f;
    if (e < p.groups) {
      v = scaled_sum(0, p.scale_a[m * p.sa_s], p.scale_b[e * p.sb_g + n * p.sb_s]);
      if (p.bias) v = __fadd_rn(v, bias_at<TO>(p, n));
    }
    static_cast<TO *>(p.C)[m * p.c_rs + n * p.c_cs] = Elem<TO>::store(v);
  }
}

}  // namespace sg
}  // namespace mb
