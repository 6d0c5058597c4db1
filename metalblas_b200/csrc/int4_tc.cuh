// Products of many tokens with 4-bit weights on tcgen05.
//
// A tile is 128 weight rows (UMMA rows, TMEM lanes) x BN tokens (UMMA columns), and
// a step 128 columns of K.  Weights come by TMA as they are, 128 rows x 256 columns
// (16 KB) a stage, are decoded to whole numbers u - z by eight warps, a thread a row
// and 64 columns, and stored to TMEM, from where the MMA reads its A operand: they
// never pass through shared memory as 16-bit values, whose writes and reads would
// bind it (the MMA of 128 x 128 takes its 128 bytes a cycle already).  Tokens come
// by TMA, BN x 128 columns a step.
//
// The MMA sums a step (a group, where groups are smaller) into one of two
// accumulators in TMEM; eight warps read it, multiply it by the row's scale, one
// number a lane, and add it to fp32 sums in registers.  So scales are applied in
// fp32 to exact products, the weights are not rounded, and the tensor core's own
// fp32 sums are short.  One tcgen05.commit a step tells the copies, the decoding and
// the sums at once (steps of 64 columns with a commit for each of them took 600 cycles
// in barriers alone).
//
// Roles, by warpgroup: warp 0 TMA, warp 1 the MMA issuer; warps 4..11 decode; warps
// 12..19 sums and output, two to a TMEM lane quarter, half of the columns each.  The
// registers go where the sums are (setmaxnreg).
// Persistent over units (matrix, token tile, row tile); units of groups are found
// in a table made from the device's offsets (int4_gemm.cuh).  A tile of tokens may
// hold rows of the next group: they are columns of their own and are not stored.
//
// split > 1 (few units): the CTAs of a cluster share a unit, each a range of
// columns of K; the warps' pieces of the tile are finished by rank piece * split / 8,
// which gets the other ranks' sums through distributed shared memory and adds
// them to its own in the order of the ranks.
//
// 4096 x 4096 x 14336: 420 us with tiles of 256 tokens, which decode a weight half as often
// (1.14 PFLOP/s; of 128 tokens 523 us; floor 292), 512 x 4096 x 4096 25.7 us.  The tensor
// pipe is in use 26 % of the latter's launch (51 % of the former's), issue slots 55 % (49 %), the logic
// pipe 45 % (38 %): decoding and sums share an SM's slots.  Groups of 64 or 32 columns have two or four sums a step, whose
// way to the registers and back binds (512 x 4096 x 4096: 37.3 and 62.7 us,
// 4096 x 4096 x 14336: 630 and 1076).
#pragma once
#include "int4_few.cuh"

namespace mb {
namespace i4 {

using namespace mb::tc;

constexpr int TC_W_BYTES = 128 * 128;    // weights of a stage: 128 rows x 256 columns
constexpr int TC_STEP = 128;             // columns of K of a step
constexpr int TC_A_COL = 256;            // first TMEM column of the weights, 64 columns a step

struct TcArgs {
  CUtensorMap w, x;
  GemmArgs g;
  int tiles_n, split, steps;             // steps of the whole of K
  int out_vec;                           // rows of out start on 16 bytes
  unsigned long long timeout_ns;
};

template <int BN> struct TcCfg {
  static constexpr int TILES = BN == 256 ? 2 : 1;   // MMAs that share a step's weights
  static constexpr int UN = BN / TILES;             // their columns
  static constexpr int STEPS = BN == 256 ? 2 : 4;   // steps held: tokens in shared memory, decoded weights in TMEM
  static constexpr int DECODERS = BN == 256 ? 4 : 8;
  static constexpr int SUM0 = 4 + DECODERS;         // first warp of the sums
  static constexpr int THREADS = (SUM0 + 8) * 32;
  // registers of a thread at launch (all of the SM's, in eights) and by role
  static constexpr int REGS = 65536 / THREADS / 8 * 8;
  static constexpr int REGS_ISSUE = 32, REGS_DECODE = BN == 256 ? 80 : 72, REGS_SUM = BN == 256 ? 192 : 152;
  static_assert(128 * REGS_ISSUE + DECODERS * 32 * REGS_DECODE + 256 * REGS_SUM <= THREADS * REGS, "registers at launch");
  static constexpr int X_TILE = UN * 128;           // a box of 64 columns
  static constexpr int X_BYTES = TILES * 2 * X_TILE;
  static constexpr int W_STAGES = BN >= 128 ? 2 : 6;
  static constexpr int D_BUFS = UN == 128 ? 2 : 4;  // accumulators
  static constexpr int CW = UN / 2;                 // columns of a warp of sums
  static constexpr int PIECE = 32 * CW * 4;         // its sums; its results are half as many bytes
  // sums from other ranks, or results on their way out
  static __host__ __device__ constexpr int red_bytes(int split) { return split > 1 ? (split - 1) * (8 / split) * PIECE : 4 * PIECE; }
  static constexpr int MAX_SPLIT = BN == 256 ? 1 : 8;
  static constexpr int NBARS = 2 * W_STAGES + 3 * STEPS + 2 * D_BUFS + 3;
  static constexpr int smem(int split, int groups) {
    return 1024 + W_STAGES * TC_W_BYTES + STEPS * X_BYTES + red_bytes(split) + (NBARS + 2) * 8 + (2 * (groups + 1) + 32) * 4;
  }
  static_assert(smem(MAX_SPLIT, kMaxGroups) <= SMEM_LIMIT, "shared memory");
};

template <int N> __device__ __forceinline__ void regs_inc() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N> __device__ __forceinline__ void regs_dec() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }
// D (+)= A B with A in TMEM.
__device__ __forceinline__ void umma_ts(uint32_t d, uint32_t a, uint64_t bdesc, uint32_t idesc, uint32_t accum) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(bdesc), "r"(idesc), "r"(accum)
      : "memory");
}
__device__ __forceinline__ void tmem_st_x32(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
      "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
      "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
      "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// The columns of a word in their order, (0, 1), (2, 3), (4, 5), (6, 7): a byte b holds
// two neighbours, and (b * 0x1001) & 0x000f000f is the pair (the multiplication
// runs beside the logic pipe, which binds the decoding).
__device__ __forceinline__ uint32_t byte_pair(uint32_t w, int i) {
  const uint32_t b = i == 0 ? w & 0xffu : i == 3 ? w >> 24 : __byte_perm(w, 0, 0x4440 + i);
  return (b * 0x1001u) & 0x000f000fu;
}
template <class T, bool ZERO> struct InOrder;
template <bool ZERO> struct InOrder<__nv_bfloat16, ZERO> {
  uint32_t z2;
  __device__ __forceinline__ explicit InOrder(uint32_t z) {
    if constexpr (ZERO) {
      const uint32_t b = __float_as_uint((float)z) >> 16;   // a whole number up to 255
      z2 = b | (b << 16);
    }
  }
  __device__ __forceinline__ void operator()(uint32_t w, uint32_t *o) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t v = byte_pair(w, i) | 0x43004300u, c = ZERO ? 0x43004300u : 0x43084308u;
      __nv_bfloat162 x = __hsub2(reinterpret_cast<const __nv_bfloat162 &>(v), reinterpret_cast<const __nv_bfloat162 &>(c));
      if constexpr (ZERO) x = __hsub2(x, reinterpret_cast<const __nv_bfloat162 &>(z2));   // 128 + z may take nine bits
      o[i] = reinterpret_cast<uint32_t &>(x);
    }
  }
};
template <bool ZERO> struct InOrder<__half, ZERO> {
  __half2 z;
  __device__ __forceinline__ explicit InOrder(uint32_t zero) {
    z = __float2half2_rn(1024.f + (ZERO ? (float)zero : 8.f));
  }
  __device__ __forceinline__ void operator()(uint32_t w, uint32_t *o) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t v = byte_pair(w, i) | 0x64006400u;
      const __half2 x = __hsub2(reinterpret_cast<const __half2 &>(v), z);
      o[i] = reinterpret_cast<const uint32_t &>(x);
    }
  }
};

struct TcTile {
  int e, r0, rend, n0;   // matrix, first token row, end of the group's rows, first weight row
};

template <class T, int BN, bool ZERO>
__global__ void __launch_bounds__(TcCfg<BN>::THREADS, 1) int4_tc_kernel(const __grid_constant__ TcArgs p) {
  using Cfg = TcCfg<BN>;
  constexpr int WS = Cfg::W_STAGES, ST = Cfg::STEPS, CW = Cfg::CW, DB = Cfg::D_BUFS, TT = Cfg::TILES, UN = Cfg::UN, ND = Cfg::DECODERS;
  const GemmArgs &a = p.g;
  const int split = p.split;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t *xring = smem + WS * TC_W_BYTES, *red = xring + ST * Cfg::X_BYTES;
  uint64_t *bars = reinterpret_cast<uint64_t *>(red + Cfg::red_bytes(split));
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(bars + Cfg::NBARS);
  volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);
  int *first_unit = reinterpret_cast<int *>(bars + Cfg::NBARS + 2);
  int *row0 = first_unit + a.groups + 1, *scan = row0 + a.groups + 1;

  // (from lane 0, so that the compiler knows it is the same for the whole warp)
  const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const uint32_t bar0 = smem_u32(bars);
  auto bar = [&](int i) { return bar0 + 8u * i; };
  // barriers: weights full, empty; a step's tokens full, its weights decoded, its MMA done;
  // an accumulator's sum done (groups below a step), read; drain, exchange
  constexpr int W_FULL = 0, W_EMPTY = WS, X_FULL = 2 * WS, A_FULL = X_FULL + ST, DONE = A_FULL + ST, D_FULL = DONE + ST,
                D_EMPTY = D_FULL + DB, DRAIN = D_EMPTY + DB, RED_FULL = DRAIN + 1, RED_FREE = DRAIN + 2;
  static_assert(RED_FREE < Cfg::NBARS, "barriers");
  const uint32_t rank = split > 1 ? cluster_rank() : 0u;
  const int cid = blockIdx.x / split, ncl = gridDim.x / split;

  pdl_trigger();
  if (threadIdx.x == 0) {
    for (int s = 0; s < WS; ++s) { mbar_init(bar(W_FULL + s), 1); mbar_init(bar(W_EMPTY + s), ND); }
    for (int s = 0; s < ST; ++s) { mbar_init(bar(X_FULL + s), 1); mbar_init(bar(A_FULL + s), ND); mbar_init(bar(DONE + s), 1); }
    for (int s = 0; s < DB; ++s) { mbar_init(bar(D_FULL + s), 1); mbar_init(bar(D_EMPTY + s), 8); }
    mbar_init(bar(DRAIN), 1);
    if (split > 1) {   // lane 0 of each sending warp; of each finishing warp
      mbar_init(bar(RED_FULL), (split - 1) * (8 / split));
      mbar_init(bar(RED_FREE), (split - 1) * (8 / split));
    }
    *abort_flag = 0;
    fence_mbar_init();
    prefetch_tmap(&p.w);
    prefetch_tmap(&p.x);
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(tmem_slot), 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  if (split > 1) cluster_sync_all();   // every CTA's barriers are initialised before any remote arrival
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);
  pdl_wait();
  // token tiles of all groups
  const int units = a.offsets ? unit_table(a, BN, first_unit, row0, scan) : (a.M + BN - 1) / BN;
  const int num_units = __shfl_sync(0xffffffffu, units * p.tiles_n, 0);
  auto unit_at = [&](int u) {
    // groups in order; within one row tiles outside, up to 16 token tiles inside (concurrent
    // CTAs share weight tiles in L2, and with many token tiles their panels too)
    TcTile t;
    int tiles_m = units, first = 0;
    t.e = 0;
    t.r0 = 0;
    t.rend = a.M;
    if (a.offsets) {
      const int g = group_of_unit(first_unit, a.groups, u / p.tiles_n);
      t.e = g;
      first = first_unit[g];
      tiles_m = first_unit[g + 1] - first;
      t.r0 = row0[g];
      t.rend = row0[g + 1];
    }
    const int v = u - first * p.tiles_n, per = 16 * p.tiles_n, grp = v / per, w = v - grp * per;
    const int gsz = min(tiles_m - grp * 16, 16);
    t.r0 += (grp * 16 + w % gsz) * BN;
    t.n0 = (w / gsz) * 128;
    return t;
  };
  // this rank's steps: whole stages of weights
  const int stages = (p.steps + 1) / 2;
  const int k0 = (int)((int64_t)rank * stages / split) * 2, k1 = min(p.steps, (int)((int64_t)(rank + 1) * stages / split) * 2);
  // sums of a step
  const int sums_log2 = max(0, 7 - a.group_log2);
  auto all = [](bool ok) { return __all_sync(0xffffffffu, ok) != 0; };

  if (warp < 4) {
    regs_dec<Cfg::REGS_ISSUE>();
    // One elected lane runs these loops: the compiler then knows that all that an instruction
    // names is uniform (with `lane == 0` every MMA had its operands moved to uniform registers
    // first and took 200 cycles to issue, whatever its size).
    if (warp == 0) {
      // ---------------------------------------------------------- producer
      if (elect_one()) {
        int ws = 0, st = 0, last_w = -1, last_x = -1;
        uint32_t wp = 0, sp = 0, last_wp = 0, last_xp = 0;
        bool ok = true;
        for (int u = cid; u < num_units && ok; u += ncl) {
          const TcTile t = unit_at(u);
          const int we = a.w_e == 0 ? 0 : t.e;
          for (int k = k0; k < k1; ++k) {
            if ((k & 1) == 0) {
              if (!mbar_wait(bar(W_EMPTY + ws), wp ^ 1u, abort_flag, p.timeout_ns)) { ok = false; break; }
              mbar_arrive_expect_tx(bar(W_FULL + ws), TC_W_BYTES);
              tma_load_3d(smem_u32(smem) + ws * TC_W_BYTES, &p.w, bar(W_FULL + ws), k * (TC_STEP / 2), t.n0, we);
              last_w = ws;
              last_wp = wp;
              if (++ws == WS) { ws = 0; wp ^= 1u; }
            }
            if (!mbar_wait(bar(DONE + st), sp ^ 1u, abort_flag, p.timeout_ns)) { ok = false; break; }
            mbar_arrive_expect_tx(bar(X_FULL + st), Cfg::X_BYTES);
            const uint32_t to = smem_u32(xring) + st * Cfg::X_BYTES;
#pragma unroll
            for (int i = 0; i < 2 * TT; ++i)   // (rows past the last token are filled with zeros)
              tma_load_3d(to + i * Cfg::X_TILE, &p.x, bar(X_FULL + st), k * TC_STEP + (i & 1) * 64, t.r0 + (i >> 1) * UN, 0);
            last_x = st;
            last_xp = sp;
            if (++st == ST) { st = 0; sp ^= 1u; }
          }
        }
        // the last copies must land before the CTA can exit
        volatile int no_abort = 0;
        if (last_w >= 0) mbar_wait(bar(W_FULL + last_w), last_wp, &no_abort, p.timeout_ns);
        if (last_x >= 0) mbar_wait(bar(X_FULL + last_x), last_xp, &no_abort, p.timeout_ns);
      }
    } else if (warp == 1) {
      // ---------------------------------------------------------- MMA issuer
      if (elect_one()) {
        const uint32_t idesc = make_idesc<T, UN>(0, 0);
        int st = 0, d = 0;
        uint32_t sp = 0, dp = 0;
        bool issued = false;
        // PER: MMAs of 16 columns in a sum.  Known here, so that a sum's MMAs follow one another: this
        // warp shares its issue slots with busy ones, and 15 instructions an MMA were 125 cycles.
        auto issue = [&](auto per) {
          constexpr int PER = decltype(per)::value;
          for (int u = cid; u < num_units; u += ncl) {
            for (int k = k0; k < k1; ++k) {
              const uint32_t at = tmem + TC_A_COL + st * 64;
              const uint64_t xd = sdesc(smem_u32(xring) + st * Cfg::X_BYTES, 16, 1024);
              if (!mbar_wait(bar(X_FULL + st), sp, abort_flag, p.timeout_ns) ||
                  !mbar_wait(bar(A_FULL + st), sp, abort_flag, p.timeout_ns))
                return;
#pragma unroll
              for (int s = 0; s < 8; s += PER) {
#pragma unroll
                for (int i = 0; i < TT; ++i) {
                  if (!mbar_wait(bar(D_EMPTY + d), dp ^ 1u, abort_flag, p.timeout_ns)) return;
                  tc_fence_after();
                  issued = true;
#pragma unroll
                  for (int ks = s; ks < s + PER; ++ks)   // (a descriptor counts shared memory in 16 bytes)
                    umma_ts(tmem + d * UN, at + ks * 8, xd + ((i * 2 + (ks >> 2)) * Cfg::X_TILE + (ks & 3) * 32) / 16, idesc, ks > s ? 1u : 0u);
                  if (PER < 8 || TT > 1) umma_commit(bar(D_FULL + d));
                  if (++d == DB) { d = 0; dp ^= 1u; }
                }
              }
              umma_commit(bar(DONE + st));
              if (++st == ST) { st = 0; sp ^= 1u; }
            }
          }
        };
        if (sums_log2 == 0) issue(std::integral_constant<int, 8>());
        else if (sums_log2 == 1) issue(std::integral_constant<int, 4>());
        else issue(std::integral_constant<int, 2>());
        if (*abort_flag && issued) {
          umma_commit(bar(DRAIN));
          volatile int no_abort = 0;
          mbar_wait(bar(DRAIN), 0, &no_abort, p.timeout_ns);
        }
      }
    }
  } else if (warp < Cfg::SUM0) {
    // ------------------------------------------------------------ decoding
    regs_dec<Cfg::REGS_DECODE>();
    constexpr int HALVES = 8 / ND;   // of a step, 64 columns each, that a thread decodes
    const int q = warp & 3, hf = ND == 8 ? (warp - 4) >> 2 : 0, r = q * 32 + lane;   // this thread's row of the tile, its TMEM lane
    const uint32_t at = tmem + TC_A_COL + hf * 32 + ((uint32_t)(q * 32) << 16);
    const uint32_t src = smem_u32(smem) + r * 128;
    int ws = 0, st = 0;
    uint32_t wp = 0, sp = 0;
    // this thread's words and zero points (of 32 columns each) of the next step
    uint4 w[2 * HALVES];
    uint32_t z[2 * HALVES];
    const uint8_t *zero = nullptr;
    auto fetch = [&](int u, int k) {
      if constexpr (ZERO) {
        if (k == k0) {
          const TcTile t = unit_at(u);
          zero = a.zero + t.e * a.z_e + (int64_t)min(t.n0 + r, a.N - 1) * a.z_rs;
        }
#pragma unroll
        for (int i = 0; i < 2 * HALVES; ++i) {
          const int c = k * TC_STEP + hf * 64 + i * 32;
          z[i] = c < a.K ? zero[c >> a.group_log2] : 8u;
        }
      }
      if ((k & 1) == 0 && !all(mbar_wait(bar(W_FULL + ws), wp, abort_flag, p.timeout_ns))) return false;
      const uint32_t row = src + ws * TC_W_BYTES;
#pragma unroll
      for (int i = 0; i < 2 * HALVES; ++i) w[i] = ld_shared_v4(row + ((((k & 1) * 4 + hf * 2 + i) ^ (r & 7)) << 4));
      if ((k & 1) || k + 1 == k1) {
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(W_EMPTY + ws));
        if (++ws == WS) { ws = 0; wp ^= 1u; }
      }
      return true;
    };
    bool ok = cid < num_units && k0 < k1 && fetch(cid, k0);
    for (int u = cid; u < num_units && ok; u += ncl) {
      for (int k = k0; k < k1; ++k) {
#pragma unroll
        for (int h = 0; h < HALVES; ++h) {
          uint32_t o[32];
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const InOrder<T, ZERO> d(ZERO ? z[2 * h + i] : 8u);
            const uint4 &v = w[2 * h + i];
            d(v.x, o + 16 * i); d(v.y, o + 16 * i + 4); d(v.z, o + 16 * i + 8); d(v.w, o + 16 * i + 12);
          }
          if (h == HALVES - 1) {
            if (k + 1 < k1) ok = fetch(u, k + 1);
            else if (u + ncl < num_units) ok = fetch(u + ncl, k0);
          }
          if (h == 0) ok = ok && all(mbar_wait(bar(DONE + st), sp ^ 1u, abort_flag, p.timeout_ns));
          if (!ok) break;
          if (h == 0) tc_fence_after();
          tmem_st_x32(at + st * 64 + h * 32, o);
        }
        if (!ok) break;
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(A_FULL + st));
        if (++st == ST) { st = 0; sp ^= 1u; }
      }
    }
  } else {
    // ------------------------------------------------------------ sums and output
    regs_inc<Cfg::REGS_SUM>();
    const int q = warp & 3, hf = (warp - Cfg::SUM0) >> 2, r = q * 32 + lane;
    T *out = static_cast<T *>(a.out);
    const int piece = q * 2 + hf, per_rank = 8 / split, owner = piece / per_rank;
    const uint32_t red_u32 = smem_u32(red) + (uint32_t)(piece % per_rank) * Cfg::PIECE + lane * 16u;
    const uint32_t red_step = (uint32_t)(per_rank * Cfg::PIECE);   // from one source rank to the next
    const int sum_log2 = min(a.group_log2, 7), end = min(a.K, k1 * TC_STEP), stop = k1 * TC_STEP;
    int d = 0, st = 0;
    uint32_t dp = 0, sp = 0, rphase = 0;
    bool first = true, ok = true;
    // the row's scales of the next AHEAD sums, as they lie in memory (converted when they are
    // used, or the first would be waited for at once)
    constexpr int AHEAD = 4;
    uint32_t next[AHEAD];
    auto fetch = [&](const TcTile &t, int k) {
      const int64_t i_s = t.e * a.s_e + (int64_t)min(t.n0 + r, a.N - 1) * a.s_rs;
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) next[i] = k + (i << sum_log2) < end ? scale_bits<T>(a, i_s + ((k + (i << sum_log2)) >> a.group_log2)) : 0u;
    };
    TcTile t, following;
    if (cid < num_units) {
      following = unit_at(cid);
      fetch(following, k0 * TC_STEP);
    }
    for (int u = cid; u < num_units && ok; u += ncl) {
      t = following;
      if (u + ncl < num_units) following = unit_at(u + ncl);
      const int64_t n = t.n0 + r;
      float acc[TT][CW];
#pragma unroll
      for (int j = 0; j < TT * CW; ++j) acc[j / CW][j % CW] = 0.f;
      for (int k = k0 * TC_STEP; k < stop && ok;) {
        float s[AHEAD];
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) s[i] = scale_of<T>(a, next[i]);
        if (k + (AHEAD << sum_log2) < stop) fetch(t, k + (AHEAD << sum_log2));
        else if (u + ncl < num_units) fetch(following, k0 * TC_STEP);
        // (not unrolled: four copies of the body missed the instruction cache)
#pragma unroll 1
        for (int i = 0; i < AHEAD && k < stop && ok; ++i, k += 1 << sum_log2) {
          const float si = i & 2 ? (i & 1 ? s[3] : s[2]) : (i & 1 ? s[1] : s[0]);
          const float2 s2 = make_float2(si, si);
#pragma unroll
          for (int tt = 0; tt < TT; ++tt) {
            if (sums_log2 || TT > 1) {
              if (!all(mbar_wait(bar(D_FULL + d), dp, abort_flag, p.timeout_ns))) { ok = false; break; }
            } else {
              if (!all(mbar_wait(bar(DONE + st), sp, abort_flag, p.timeout_ns))) { ok = false; break; }
              if (++st == ST) { st = 0; sp ^= 1u; }
            }
            tc_fence_after();
            const uint32_t from = tmem + ((uint32_t)(q * 32) << 16) + d * UN + hf * CW;
            constexpr int CH = CW < 32 ? CW : 32;
#pragma unroll
            for (int c = 0; c < CW; c += CH) {
              uint32_t v[32];
              tmem_ld<CH>(from + c, v);
              tmem_wait_ld();
              if (c + CH >= CW) {   // the accumulator is read
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(bar(D_EMPTY + d));
              }
#pragma unroll
              for (int j = 0; j < CH; j += 2) {
                const float2 o = fma2(make_float2(__uint_as_float(v[j]), __uint_as_float(v[j + 1])), s2,
                                      make_float2(acc[tt][c + j], acc[tt][c + j + 1]));
                acc[tt][c + j] = o.x;
                acc[tt][c + j + 1] = o.y;
              }
            }
            if (++d == DB) { d = 0; dp ^= 1u; }
          }
        }
      }
      if (!ok) break;
      if (Cfg::MAX_SPLIT > 1 && split > 1) {
        if (owner != (int)rank) {
          // what this CTA sent for the last unit has been read
          if (!first && !all(mbar_wait_cluster(bar(RED_FREE), rphase ^ 1u, abort_flag, p.timeout_ns))) break;
          const uint32_t dst = mapa_shared(red_u32 + (uint32_t)((int)rank - ((int)rank > owner ? 1 : 0)) * red_step, (uint32_t)owner);
#pragma unroll
          for (int j = 0; j < CW; j += 4)
            st_cluster_v4(dst + (uint32_t)(j >> 2) * 512u, __float_as_uint(acc[0][j]), __float_as_uint(acc[0][j + 1]),
                          __float_as_uint(acc[0][j + 2]), __float_as_uint(acc[0][j + 3]));
          __syncwarp();   // the lanes' stores come before lane 0's release
          if (lane == 0) mbar_arrive_cluster(mapa_shared(bar(RED_FULL), (uint32_t)owner));
        } else {
          if (!all(mbar_wait_cluster(bar(RED_FULL), rphase, abort_flag, p.timeout_ns))) break;
          // to this rank's own sums, in the order of the ranks
#pragma unroll 1
          for (int s = 0; s < split - 1; ++s) {
#pragma unroll
            for (int j = 0; j < CW; j += 4) {
              const uint4 v = ld_shared_v4(red_u32 + s * red_step + (uint32_t)(j >> 2) * 512u);
              acc[0][j] += __uint_as_float(v.x);
              acc[0][j + 1] += __uint_as_float(v.y);
              acc[0][j + 2] += __uint_as_float(v.z);
              acc[0][j + 3] += __uint_as_float(v.w);
            }
          }
        }
      }
      if (split == 1 || owner == (int)rank) {
        // Lanes hold rows of the weights, columns of the output: transposed through this warp's own
        // shared memory (its sums of the other ranks have been read), so that rows leave in
        // whole 16 bytes where they lie on them.
        const float b = a.bias && n < a.N ? bias_at<T>(a, n) : 0.f;
        T *stage = reinterpret_cast<T *>(split > 1 ? red + (piece % per_rank) * Cfg::PIECE : red + piece * (Cfg::PIECE / 2));
        const int64_t nw = t.n0 + q * 32;
#pragma unroll
        for (int tt = 0; tt < TT; ++tt) {
          __syncwarp();
#pragma unroll
          for (int j = 0; j < CW; ++j) stage[j * 32 + lane] = Elem<T>::store(acc[tt][j] + b);
          __syncwarp();
          const int64_t m = t.r0 + tt * UN + hf * CW;
          const int live = (int)max((int64_t)0, min((int64_t)CW, t.rend - m));
          T *dst = out + m * a.out_rs + nw;
          if (p.out_vec && nw + 32 <= a.N) {
            for (int j = lane >> 2; j < live; j += 8)
              *reinterpret_cast<uint4 *>(dst + j * a.out_rs + (lane & 3) * 8) = *reinterpret_cast<const uint4 *>(stage + j * 32 + (lane & 3) * 8);
          } else if (n < a.N) {
            for (int j = 0; j < live; ++j) dst[j * a.out_rs + lane] = stage[j * 32 + lane];
          }
        }
        if (split > 1) {
          __syncwarp();
          if (lane < split && lane != (int)rank) mbar_arrive_cluster(mapa_shared(bar(RED_FREE), (uint32_t)lane));
        }
      }
      rphase ^= 1u;
      first = false;
    }
    if (a.offsets) zero_rest<T>(a, row0[a.groups], threadIdx.x - Cfg::SUM0 * 32, 8 * 32);
  }

  tc_fence_before();
  __syncthreads();
  if (split > 1) cluster_sync_all();   // no CTA leaves while others still reach its shared memory
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_g<1>(tmem, 512);
  }
}

}  // namespace i4
}  // namespace mb
