// C ABI of the int8 products with scales (quantize.cuh, scaled_tc.cuh,
// scaled_gemv.cuh) and of the expert routing (experts.cuh).
#include <cuda.h>
#include <cuda_runtime.h>

#include <atomic>
#include <cmath>
#include <cstring>
#include <numeric>
#include <type_traits>

#include "mb_host.cuh"
#include "mb_common.cuh"
#include "quantize.cuh"
#include "experts.cuh"
#include "pack.cuh"
#include "scaled_tc.cuh"
#include "scaled_gemv.cuh"

using namespace mb;
using namespace mb::host;

int mb::ops_status_read(int *v) {
  return cuda_check(cudaMemcpyFromSymbol(v, g_mb_status, sizeof(int)), "read status");
}
void mb::ops_status_clear() {
  int z = 0;
  cudaMemcpyToSymbol(g_mb_status, &z, sizeof(int));
}

namespace {

// f(tag) with a null pointer of the element type of a float dtype.
template <class F>
int by_float(int dt, F &&f) {
  switch (dt) {
    case MB_F32: return f((float *)nullptr);
    case MB_F16: return f((__half *)nullptr);
    case MB_BF16: return f((__nv_bfloat16 *)nullptr);
  }
  return fail(MB_ERR_UNSUPPORTED, "dtype %d is not a float type of this function (fp32, fp16, bf16)", dt);
}
bool is_float(int dt) { return dt == MB_F32 || dt == MB_F16 || dt == MB_BF16; }

// Every row of the buffer starts on a 16-byte boundary.
bool rows16(const void *p, int64_t ld, int esz) { return aligned16(p) && (ld * esz) % 16 == 0; }

int check_rows(int dt, int64_t rows, int64_t cols, int64_t ld, const void *p, const char *what) {
  if (rows < 0 || cols < 0) return fail(MB_ERR_INVALID, "%s: negative extent", what);
  if (cols > (1ll << 30)) return fail(MB_ERR_INVALID, "%s: %lld columns", what, (long long)cols);
  if (rows > 1 && ld < cols) return fail(MB_ERR_INVALID, "%s: row stride %lld below %lld columns", what, (long long)ld, (long long)cols);
  if (rows > 0 && cols > 0 && !p) return fail(MB_ERR_INVALID, "%s: null pointer", what);
  return MB_OK;
}

int check_route(int64_t T, int64_t k, int64_t H, const int32_t *position, const int32_t *kept) {
  if (T < 0 || k < 0 || H < 0) return fail(MB_ERR_INVALID, "negative extent");
  if (T > 0x7fff0000ll || (k && T > 0x7fff0000ll / k)) return fail(MB_ERR_INVALID, "tokens * k must stay below 2^31 - 2^16");
  if (T * k > 0 && (!position || !kept)) return fail(MB_ERR_INVALID, "null position or kept");
  return MB_OK;
}


// Threads of a block that share a token: short rows would leave most of a block idle.
int route_lanes(int64_t H, int esz, bool whole_warps) {
  const int64_t vecs = ceil_div(H * esz, 16);
  if (!whole_warps && vecs <= 16) return 16;
  return vecs <= 64 ? 32 : vecs <= 512 ? 128 : 256;
}
dim3 route_grid(int64_t T, int64_t H, int esz, int lanes, bool whole_rows) {
  const int64_t x = ceil_div(T, kRouteThreads / lanes);
  // with few tokens a row is shared out as far as its vectors go
  int64_t y = whole_rows ? 1 : std::min<int64_t>(ceil_div(ceil_div(H * esz, 16) + 1, lanes), 64);
  y = std::min<int64_t>(y, std::max<int64_t>(1, ceil_div(16 * (int64_t)device_sms(), x)));
  return dim3((unsigned)x, (unsigned)y);
}

constexpr size_t sort_smem(int warps, int64_t experts) {
  return ((size_t)warps * ((experts + 1) | 1) + experts + 1 + 32) * 4;
}
// Sets the sort kernel up on the current device, once: its largest shared memory,
// and whether the device runs clusters of 16 of its largest blocks (past the
// portable 8).
template <class I>
int sort_setup(int &max_ranks) {
  static std::atomic<int> ranks[64];
  int dev = 0;
  int rc = cuda_check(cudaGetDevice(&dev), "cudaGetDevice");
  if (rc) return rc;
  const bool keep = dev >= 0 && dev < 64;
  if (keep && (max_ranks = ranks[dev].load(std::memory_order_acquire)) > 0) return MB_OK;
  auto kern = expert_sort_kernel<I>;
  const size_t smem = sort_smem(32, kMaxExperts);
  rc = cuda_check(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem), "cudaFuncSetAttribute");
  if (rc) return rc;
  max_ranks = 8;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(kSortRanks);
  cfg.blockDim = dim3(1024);
  cfg.dynamicSmemBytes = smem;
  cudaLaunchAttribute a[1];
  a[0].id = cudaLaunchAttributeClusterDimension;
  a[0].val.clusterDim.x = kSortRanks;
  a[0].val.clusterDim.y = a[0].val.clusterDim.z = 1;
  cfg.attrs = a;
  cfg.numAttrs = 1;
  int clusters = 0;
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) == cudaSuccess &&
      cudaOccupancyMaxActiveClusters(&clusters, kern, &cfg) == cudaSuccess && clusters > 0)
    max_ranks = kSortRanks;
  (void)cudaGetLastError();
  if (keep) ranks[dev].store(max_ranks, std::memory_order_release);
  return MB_OK;
}

template <class T>
int launch_quantize(const RouteParams &p, cudaStream_t st, const char *what) {
  constexpr int V = Vec<T>::V;
  const bool al = rows16(p.src, p.ld_src, sizeof(T));
  const int q_vec = reinterpret_cast<uintptr_t>(p.dst) % V == 0 && p.ld_dst % V == 0;
  const int64_t vecs = ceil_div(p.H, V);
  auto go = [&](auto tpr_, auto held_) {
    constexpr int TPR = decltype(tpr_)::value, HELD = decltype(held_)::value, threads = TPR < 256 ? 256 : TPR;
    auto kern = al ? quantize_rows_kernel<T, true, TPR, HELD> : quantize_rows_kernel<T, false, TPR, HELD>;
    return launch_pdl(kern, dim3((unsigned)ceil_div(p.T, threads / TPR)), dim3(threads), 0, st, 1, what, p, q_vec);
  };
  using std::integral_constant;
  // Threads to a row and vectors they hold, by the row's vectors, measured on B200
  // with 2, 4 and 8 held: many rows want them held by few threads (16384 x 4096
  // bf16 41.5 us by 128, 44.3 by 256; 8192 x 14336 70 us by 256, 88 by 512), few
  // rows want many threads (1024 x 4096 3.9 us by 256, 4.5 by 128).  A row between
  // two sizes leaves slots empty whose instructions are issued all the same: 7601 x
  // 5408, 676 vectors of 1024, 30.2 us, 141 warp instructions for 256 elements (116
  // at 16384 x 8192) with the issue slots 73 % in use.
  if (vecs <= 16) return go(integral_constant<int, 8>(), integral_constant<int, 2>());
  if (vecs <= 64) return go(integral_constant<int, 32>(), integral_constant<int, 2>());
  if (vecs <= 128) return go(integral_constant<int, 32>(), integral_constant<int, 4>());
  if (vecs <= 256) return go(integral_constant<int, 128>(), integral_constant<int, 2>());
  if (vecs <= 512 && p.T < 4096) return go(integral_constant<int, 256>(), integral_constant<int, 2>());
  if (vecs <= 512) return go(integral_constant<int, 128>(), integral_constant<int, 4>());
  if (vecs <= 1024) return go(integral_constant<int, 256>(), integral_constant<int, 4>());
  if (vecs <= 2048 && p.T < 512) return go(integral_constant<int, 512>(), integral_constant<int, 4>());
  if (vecs <= 2048) return go(integral_constant<int, 256>(), integral_constant<int, 8>());
  return go(integral_constant<int, 512>(), integral_constant<int, 8>());
}

// ------------------------------------------------------------- int8 products with scales
// Whether two elements of a rows x cols matrix have one address: i rs + j cs = 0
// for some |i| < rows and |j| < cols, not both 0.  The least such pair is the
// strides over their greatest common divisor.
bool share_memory(int64_t rows, int64_t cols, int64_t rs, int64_t cs) {
  if (rows <= 1) return cols > 1 && cs == 0;
  if (cols <= 1) return rs == 0;
  rs = std::abs(rs);
  cs = std::abs(cs);
  const int64_t g = std::gcd(rs, cs);
  return g == 0 || (cs / g < rows && rs / g < cols);
}
int scaled_check(const mb_scaled_desc *d) {
  if (!d) return fail(MB_ERR_INVALID, "null descriptor");
  if (!is_float(d->out_dtype)) return fail(MB_ERR_UNSUPPORTED, "out_dtype %d is not fp32, fp16 or bf16", d->out_dtype);
  if (d->M < 0 || d->N < 0 || d->K < 0 || d->groups < 0) return fail(MB_ERR_INVALID, "negative extent");
  if (d->M > 0x7fff0000ll || d->N > 0x7fff0000ll) return fail(MB_ERR_INVALID, "M and N must stay below 2^31 - 2^16");
  if (d->K > 131071) return fail(MB_ERR_INVALID, "K = %lld: sums of more than 131071 int8 products can leave 32 bits", (long long)d->K);
  if (d->groups > 1024) return fail(MB_ERR_INVALID, "more than 1024 groups");
  if (d->M == 0 || d->N == 0) return MB_OK;
  if (!d->C || !d->scale_a || !d->scale_b) return fail(MB_ERR_INVALID, "null C, scale_a or scale_b");
  if (share_memory(d->M, d->N, d->c_rs, d->c_cs))
    return fail(MB_ERR_INVALID, "elements of C share memory (strides %lld, %lld)", (long long)d->c_rs, (long long)d->c_cs);
  if (d->K > 0 && (!d->A || !d->B)) return fail(MB_ERR_INVALID, "null A or B");
  if (d->groups > 0 && !d->offsets) return fail(MB_ERR_INVALID, "groups need offsets");
  if (d->bias && d->bias_dtype != d->out_dtype && d->bias_dtype != MB_F32)
    return fail(MB_ERR_INVALID, "bias must have the output's type or fp32");
  return MB_OK;
}


struct SgPlan {
  bool empty = false;
  bool gemv = false;                  // one row, or few by group: one pass over the weights
  int thin = 0;                       // two to sixteen rows: the same; blocks per SM
  int bn = 0, pair = 1, split = 1, swap = 0;
  int w_mn = 0;                       // weights are read with N contiguous
  int pk_a = 0, pk_b = 0;             // operand copied into the workspace first
  int64_t a_rs = 0, w_ld = 0, sB = 0; // strides of the operands as read
  int64_t a_off = 0, b_off = 0, ws_bytes = 0;
  int64_t units = 0;                  // at most
};

// TMA reads a matrix in place when `cs` is 1, the base lies on 16 bytes and rows
// (and groups) are a multiple of 16 bytes apart.
bool tma_rows(const void *p, int64_t rows, int64_t cols, int64_t &rs, int64_t cs, int64_t groups, int64_t gs) {
  if (cols > 1 && cs != 1) return false;
  if (rows <= 1) rs = round_up(std::max<int64_t>(cols, 1), 16);  // never used to step
  return aligned16(p) && rs > 0 && rs % 16 == 0 && (groups <= 1 || (gs >= 0 && gs % 16 == 0));
}

// One tile shape's time in SM cycles.  A tile takes its 128-byte K-blocks and a
// hand-over; beside it runs the epilogue of the tile before, so a wave takes the
// longer of the two, and the last wave both.  The chip's HBM gives 22.4 B/clk per
// SM.  Splitting K costs a cluster's exchange for each doubling.  The constants are
// fitted to times on B200 of every tile and split over 240 shapes (17 to 16000
// rows, K of 128 to 12000, N of 256 to 15000, half as many with 4 to 128 groups): the
// choice costs 2% over the best tile in the mean (7% with a model that had the
// last wave's epilogue run beside the next).  A 512-wide pair tile won in none.
struct SgCost {
  double t;
  int split;
};
SgCost sg_cost(const mb_scaled_desc *d, int swap, int bn, int pair, int sms, int force_split) {
  const double M = (double)d->M, kb = (double)ceil_div(d->K, 128);
  const double active = d->groups ? std::min<double>((double)d->groups, M) : 1.0;
  const double rows = M / active;
  const int trows = swap ? bn : 128 * pair;
  // groups do not end on tile boundaries: half a tile more each
  const double tiles_r = d->groups && rows > trows / 2 ? M / trows + 0.5 * active : active * std::ceil(rows / trows);
  const double units = tiles_r * (double)ceil_div(d->N, swap ? 128 : bn);
  const double kbc = pair == 2 ? 660.0 : bn == 256 ? 850.0 : (128.0 + bn) * 128.0 / (swap ? 46.5 : 49.5);
  const double hand = pair == 2 ? 2560.0 : bn == 256 ? 2900.0 : 1200.0;
  const double epi = pair == 2 ? 10400.0 : (swap ? 37.5 : bn == 256 ? 19.7 : 29.5) * bn;
  const double start = pair == 2 ? 2600.0 : bn == 256 ? 2150.0 : swap ? 5100.0 : 2950.0;
  // a group's weights read for a second tile of its rows come from L2, mostly
  const double again = d->groups ? 0.14 * std::min(1.0, tiles_r / active - 1.0) : 0.0;
  const double bytes = active * (double)d->N * (double)d->K * (1.0 + again) + M * (double)d->K +
                       M * (double)d->N * elem_size(d->out_dtype);
  SgCost best{1e300, 1};
  for (int split = 1, log2 = 0; split <= 8; split *= 2, ++log2) {
    if (force_split ? split != force_split : (split > 1 && (pair == 2 || bn > 128 || kb < split))) continue;
    // clusters of 4 and 8 leave SMs over in some GPCs
    const double slots = std::floor((double)sms / (pair * split) * (split == 8 ? 0.75 : split == 4 ? 0.9 : 1.0));
    const double waves = std::ceil(units / slots);
    const double tile = std::ceil(kb / split) * kbc + hand + log2 * 1960.0;
    const double compute = start + (waves - 1.0) * std::max(tile, epi) + tile + epi;
    const double hbm = bytes / (22.4 * sms);
    const double t = std::max(compute, hbm) + 0.35 * std::min(compute, hbm);  // they overlap, not quite
    if (t < best.t) best = {t, split};
  }
  return best;
}

// The single-pass kernel's weight rows of a block, at most, and its shared memory.
int64_t gemv_max_rows(const mb_scaled_desc *d) {
  const int64_t total = (d->groups ? d->M : 1) * d->N;
  return ceil_div(total, (int64_t)device_sms() * sg::GEMV_BLOCKS_PER_SM) + 1;
}
int64_t gemv_smem(const mb_scaled_desc *d) {
  const int64_t mr = d->groups ? 1 : d->M;
  return d->M * round_up(d->K, 16) + gemv_max_rows(d) * mr * 4;
}
constexpr int kGemvSmem = 96 * 1024;  // two blocks to an SM
int64_t thin_max_rows(const mb_scaled_desc *d, int per_sm) { return ceil_div(d->N, (int64_t)device_sms() * per_sm); }
int64_t thin_smem(const mb_scaled_desc *d, int per_sm) {
  return (d->M > 8 ? 16 : 8) * (int64_t)(sg::thin_pitch((int)d->K) + 4 * sg::thin_sums((int)thin_max_rows(d, per_sm)));
}
constexpr int kThinSmem = 216 * 1024;

int sg_plan(const mb_scaled_desc *d, SgPlan &pl) {
  if (d->M == 0 || d->N == 0) { pl.empty = true; return MB_OK; }
  if (d->K == 0) return MB_OK;
  const int64_t E = std::max<int64_t>(d->groups, 1);
  const int64_t nB = d->groups > 1 && d->sB == 0 ? 1 : E;  // distinct weight matrices
  // tokens: K contiguous
  pl.a_rs = d->a_rs;
  if (!tma_rows(d->A, d->M, d->K, pl.a_rs, d->a_cs, 1, 0)) {
    pl.pk_a = 1;
    pl.a_rs = round_up(d->K, 16);
  }
  // weights: K or N contiguous, as they come; without a unit stride copied with K contiguous
  pl.w_ld = d->b_cs;
  pl.sB = d->sB;
  if (!tma_rows(d->B, d->N, d->K, pl.w_ld, d->b_rs, nB, d->sB)) {
    pl.w_ld = d->b_rs;
    pl.w_mn = 1;
    if (!tma_rows(d->B, d->K, d->N, pl.w_ld, d->b_cs, nB, d->sB)) {
      pl.pk_b = 1;
      pl.w_mn = d->b_cs == 1 && d->b_rs != 1;
      pl.w_ld = round_up(pl.w_mn ? d->N : d->K, 16);
      pl.sB = pl.w_ld * (pl.w_mn ? d->K : d->N);
    }
  }
  int64_t at = 0;
  if (pl.pk_a) { pl.a_off = at; at = round_up(at + d->M * pl.a_rs, 256); }
  if (pl.pk_b) { pl.b_off = at; at = round_up(at + nB * pl.sB, 256); }
  pl.ws_bytes = at;

  const int sms = device_sms();
  const bool forced = d->tile_n || d->cta_pair || d->split_k || d->swap_ab;
  if (!forced && !pl.pk_a && !pl.pk_b && !pl.w_mn) {
    // Few rows: one of the single-pass kernels of scaled_gemv.cuh, by the weights'
    // bytes.  The MMA one starts first (4 x 2048 x 1536 3.5 us, tcgen05 5.1) but streams
    // at 4.5 TB/s; the dp4a one streams two rows faster and starts later.  MMA kernel
    // against what runs otherwise (two rows: dp4a, more: tcgen05), us at so many MiB:
    //   K = 4096   2 rows   16: 5.7, 5.7    20: 7.1, 6.3    24: 8.0, 7.7
    //              4 rows   32: 8.9, 11.4   40: 12.2, 13.2  48: 13.4, 13.6  64: 16.4, 15.0
    //              16 rows  16: 7.5, 8.8    20: 8.9, 10.3   24: 9.8, 10.3   40: 14.1, 13.5
    //   K = 1024   2 rows   8: 4.3, 3.5     16: 6.3, 4.4
    //              4 rows   8: 4.3, 5.3     16: 6.5, 6.4    24: 8.8, 8.0    40: 13.2, 11.0
    //              16 rows  8: 4.9, 5.3     16: 7.3, 6.5    20: 9.0, 7.8
    //   K = 12288  2 rows   8: 10.5, 5.1    16: 12.0, 5.9
    //              4 rows   8: 10.9, 7.7    40: 19.6, 13.6
    // The limits fit K near 4096.  With rows of 1 KB the MMA kernel's range ends
    // earlier, and at K = 12288 it is slower at every size: the bytes alone do not tell.
    const int64_t weights = d->K * d->N, small = (d->M > 8 || d->M == 2 ? 20ll : 40ll) << 20;
    if (!d->groups && d->M > 1 && d->M <= sg::THIN_ROWS && weights <= small) {
      pl.thin = thin_smem(d, 2) <= kThinSmem / 2 ? 2 : thin_smem(d, 1) <= kThinSmem ? 1 : 0;
      if (pl.thin) return MB_OK;
    }
    if (d->M <= (d->groups ? sg::GEMV_GROUPED_ROWS : sg::GEMV_ROWS) && gemv_smem(d) <= kGemvSmem) {
      pl.gemv = true;
      return MB_OK;
    }
  }
  static const struct { int swap, bn, pair; } tiles[] = {{1, 16, 1},  {1, 32, 1},  {1, 64, 1},  {1, 128, 1},
                                                         {0, 128, 1}, {0, 256, 1}, {0, 256, 2}};
  double best = 1e300;
  for (const auto &c : tiles) {
    if (d->tile_n && d->tile_n != c.bn) continue;
    if (d->cta_pair && d->cta_pair != c.pair) continue;
    if (d->swap_ab && (d->swap_ab > 0) != (c.swap == 1)) continue;
    if (d->split_k > 1 && (c.pair != 1 || c.bn > 128)) continue;
    const SgCost cost = sg_cost(d, c.swap, c.bn, c.pair, sms, d->split_k);  // (an impossible split: never less)
    if (cost.t < best) {
      best = cost.t;
      pl.swap = c.swap; pl.bn = c.bn; pl.pair = c.pair; pl.split = cost.split;
    }
  }
  if (!pl.bn) return fail(MB_ERR_INVALID, "no tile has tile_n %d, split_k %d, swap_ab %d, cta_pair %d", d->tile_n, d->split_k, d->swap_ab, d->cta_pair);
  if (pl.split != 1 && pl.split != 2 && pl.split != 4 && pl.split != 8)
    return fail(MB_ERR_INVALID, "split_k must be 1, 2, 4 or 8");
  if (pl.split > ceil_div(d->K, 128)) return fail(MB_ERR_INVALID, "split_k %d exceeds the K-blocks", pl.split);
  const int64_t trows = pl.swap ? pl.bn : 128 * pl.pair;
  pl.units = (ceil_div(d->M, trows) + (d->groups ? std::min(E, d->M) : 0)) * ceil_div(d->N, pl.swap ? 128 : pl.bn);
  if (pl.units >= (1ll << 31)) return fail(MB_ERR_INVALID, "too many tiles");
  return MB_OK;
}

template <int MR, bool GROUPED, int ROWSTEPS, class TO>
int gemv_launch_as(const mb_scaled_desc *d, const SgPlan &pl, const sg::SgParams &p, cudaStream_t st) {
  sg::GemvArgs g{};
  g.A = d->A; g.B = d->B; g.a_rs = pl.a_rs; g.b_rs = pl.w_ld; g.sB = pl.sB;
  g.K = (int)d->K;
  g.max_rows = (int)gemv_max_rows(d);
  constexpr auto kern = sg::scaled_gemv_kernel<MR, GROUPED, ROWSTEPS, TO>;
  const int rc = allow_smem<kern>(kGemvSmem);
  if (rc) return rc;
  return launch_pdl(kern, dim3((unsigned)(device_sms() * sg::GEMV_BLOCKS_PER_SM)), dim3(sg::GEMV_THREADS),
                    (size_t)gemv_smem(d), st, 1, "scaled_gemm", p, g);
}
// Rows are taken whole when they are short and every warp has some.
template <int MR, bool GROUPED, class TO>
int gemv_launch(const mb_scaled_desc *d, const SgPlan &pl, const sg::SgParams &p, cudaStream_t st) {
  const int64_t warps = (int64_t)device_sms() * sg::GEMV_BLOCKS_PER_SM * (sg::GEMV_THREADS / 32);
  const bool whole = (d->groups ? d->M : 1) * d->N > warps;
  if (whole && d->K <= 512) return gemv_launch_as<MR, GROUPED, 1, TO>(d, pl, p, st);
  if (whole && d->K <= 1024) return gemv_launch_as<MR, GROUPED, 2, TO>(d, pl, p, st);
  if (whole && d->K <= 2048) return gemv_launch_as<MR, GROUPED, 4, TO>(d, pl, p, st);
  return gemv_launch_as<MR, GROUPED, 0, TO>(d, pl, p, st);
}

template <bool MANY, class TO>
int thin_launch(const mb_scaled_desc *d, const SgPlan &pl, const sg::SgParams &p, cudaStream_t st) {
  sg::GemvArgs g{};
  g.A = d->A; g.B = d->B; g.a_rs = pl.a_rs; g.b_rs = pl.w_ld;
  g.K = (int)d->K;
  g.max_rows = (int)thin_max_rows(d, pl.thin);
  constexpr auto kern = sg::scaled_thin_kernel<MANY, TO>;
  const int rc = allow_smem<kern>(kThinSmem);
  if (rc) return rc;
  return launch_pdl(kern, dim3((unsigned)(device_sms() * pl.thin)), dim3(sg::THIN_THREADS), (size_t)thin_smem(d, pl.thin),
                    st, 1, "scaled_gemm", p, g);
}

template <int BN, int PAIR, bool SWAP, class TO, bool RUNS = false>
int sg_launch_tile(const SgPlan &pl, sg::SgParams &p, cudaStream_t st) {
  if constexpr (!SWAP && !RUNS) {
    if (!p.c_vec && p.c_cs == 1) return sg_launch_tile<BN, PAIR, SWAP, TO, true>(pl, p, st);
  }
  using C_ = sg::SgCfg<BN, PAIR, SWAP, TO>;
  p.split = pl.split;
  p.stages = C_::stages(pl.split);
  p.tiles_c = (int)ceil_div(p.N, C_::TCOLS);
  constexpr auto kern = sg::scaled_gemm_kernel<BN, PAIR, SWAP, RUNS, TO>;
  constexpr int smem_max = C_::CAN_SPLIT ? std::max(C_::smem_bytes(1), std::max(C_::smem_bytes(2), std::max(C_::smem_bytes(4), C_::smem_bytes(8))))
                                         : C_::smem_bytes(1);
  static_assert(smem_max <= tc::SMEM_LIMIT, "shared memory");
  const int rc = allow_smem<kern>(smem_max);
  if (rc) return rc;
  const int csize = PAIR == 2 ? 2 : pl.split;
  const int64_t clusters = std::min<int64_t>(pl.units, device_sms() / csize);
  return launch_pdl(kern, dim3((unsigned)(clusters * csize)), dim3(tc::NUM_THREADS), C_::smem_bytes(pl.split), st, csize,
                    "scaled_gemm", p);
}

// Copies the operands that need it (rows of neither: null).  Rows go sixteen
// bytes a thread, of groups with rows (offsets: as p.offsets, b's batches the
// groups) alone; a matrix without a unit stride through tiles.
int sg_pack(const PackArgs *a, const PackArgs *b, const int *offsets, int M, cudaStream_t st) {
  const int64_t cap = (int64_t)device_sms() * 16;
  for (const PackArgs **m : {&a, &b}) {
    if (!*m || (*m)->cs == 1) continue;
    const int64_t tiles = (*m)->batch * ceil_div((*m)->rows, 32) * ceil_div((*m)->cols, 32);
    pack_matrix_kernel<uint8_t><<<(unsigned)std::min<int64_t>(tiles, cap), dim3(32, 8), 0, st>>>(**m);
    const int rc = cuda_check(cudaGetLastError(), "scaled_gemm: operand copy");
    if (rc) return rc;
    *m = nullptr;
  }
  auto blocks = [&](const PackArgs *m) {
    return m ? std::min<int64_t>(ceil_div(m->batch * m->rows * ceil_div(m->cols, 512), 8), (int64_t)device_sms() * 4) : 0;
  };
  const int64_t na = blocks(a), nb = blocks(b);
  if (na + nb == 0) return MB_OK;
  const PackArgs none{};
  return launch_pdl(sg::scaled_pack_kernel, dim3((unsigned)(na + nb)), dim3(256), 0, st, 1, "scaled_gemm: operand copy",
                    a ? *a : none, b ? *b : none, (int)na, offsets, M);
}

template <class TO>
int sg_launch(const mb_scaled_desc *d, const SgPlan &pl, cudaStream_t st) {
  sg::SgParams p;
  memset(&p, 0, sizeof(p));
  p.M = (int)d->M; p.N = (int)d->N; p.groups = (int)std::max<int64_t>(d->groups, 1);
  p.offsets = d->groups ? d->offsets : nullptr;
  p.one_b = d->groups > 1 && d->sB == 0;
  p.K = (int)d->K;
  p.kb_total = (int)ceil_div(d->K, 128);
  p.C = d->C; p.c_rs = d->c_rs; p.c_cs = d->c_cs;
  constexpr int OSZ = sizeof(TO);
  p.c_vec = (d->c_cs == 1 || d->N == 1) && aligned16(d->C) && (d->M == 1 || (d->c_rs * OSZ) % 16 == 0);
  p.scale_a = d->scale_a; p.scale_b = d->scale_b;
  p.sa_s = d->scale_a_s; p.sb_s = d->scale_b_s; p.sb_g = d->scale_b_g;
  p.bias = d->bias; p.bias_s = d->bias_s; p.bias_f32 = d->bias_dtype == MB_F32;
  p.timeout_ns = wait_timeout_ns();
  if (d->K == 0) {
    const int64_t blocks = std::min<int64_t>(ceil_div(d->M * d->N, 256), (int64_t)device_sms() * 16);
    return launch_pdl(sg::scaled_empty_kernel<TO>, dim3((unsigned)blocks), dim3(256), 0, st, 1, "scaled_gemm", p);
  }
  if (pl.gemv) {
    if (d->groups) return gemv_launch<1, true, TO>(d, pl, p, st);
    return d->M == 1 ? gemv_launch<1, false, TO>(d, pl, p, st) : gemv_launch<2, false, TO>(d, pl, p, st);
  }
  if (pl.thin) return d->M > 8 ? thin_launch<true, TO>(d, pl, p, st) : thin_launch<false, TO>(d, pl, p, st);
  const int64_t nB = p.one_b ? 1 : p.groups;
  const void *A = d->A, *B = d->B;
  PackArgs pa{}, pb{};
  if (pl.pk_a) {
    A = static_cast<char *>(d->workspace) + pl.a_off;
    pa = PackArgs{d->A, const_cast<void *>(A), d->M, d->K, d->a_rs, d->a_cs, 0, 1, pl.a_rs};
  }
  if (pl.pk_b) {
    B = static_cast<char *>(d->workspace) + pl.b_off;
    pb = pl.w_mn ? PackArgs{d->B, const_cast<void *>(B), d->K, d->N, d->b_rs, d->b_cs, d->sB, nB, pl.w_ld}
                 : PackArgs{d->B, const_cast<void *>(B), d->N, d->K, d->b_cs, d->b_rs, d->sB, nB, pl.w_ld};
  }
  int rc = sg_pack(pl.pk_a ? &pa : nullptr, pl.pk_b ? &pb : nullptr, p.one_b ? nullptr : p.offsets, p.M, st);
  if (rc) return rc;
  // boxes of 128 bytes along the contiguous dimension
  CUtensorMap *ta = pl.swap ? &p.tmB : &p.tmA, *tw = pl.swap ? &p.tmA : &p.tmB;
  const int w_rows = pl.swap ? 128 : pl.bn / pl.pair;  // channels per box
  rc = encode_map(ta, MB_I8, A, d->K, d->M, 1, pl.a_rs, 0, 128, pl.swap ? pl.bn : 128);
  if (!rc)
    rc = pl.w_mn ? encode_map(tw, MB_I8, B, d->N, d->K, nB, pl.w_ld, pl.sB, 128, 128)
                 : encode_map(tw, MB_I8, B, d->K, d->N, nB, pl.w_ld, pl.sB, 128, w_rows);
  if (rc) return rc;
  (pl.swap ? p.a_mn : p.b_mn) = pl.w_mn;
  if (!pl.swap && p.c_vec && (d->M == 1 || d->c_rs >= d->N))
    p.c_tma = encode_map(&p.tmC, d->out_dtype, d->C, d->N, d->M, 1, d->M == 1 ? round_up(d->N, 16) : d->c_rs, 0, 32, 32,
                         OSZ == 4 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B) == MB_OK;
  if (pl.swap && !d->groups && !pl.w_mn) {
    p.w = static_cast<const int8_t *>(B);
    p.w_ld = pl.w_ld;
  }
  if (pl.swap) {
    switch (pl.bn) {
      case 16: return sg_launch_tile<16, 1, true, TO>(pl, p, st);
      case 32: return sg_launch_tile<32, 1, true, TO>(pl, p, st);
      case 64: return sg_launch_tile<64, 1, true, TO>(pl, p, st);
      default: return sg_launch_tile<128, 1, true, TO>(pl, p, st);
    }
  }
  if (pl.pair == 1) return pl.bn == 128 ? sg_launch_tile<128, 1, false, TO>(pl, p, st) : sg_launch_tile<256, 1, false, TO>(pl, p, st);
  return sg_launch_tile<256, 2, false, TO>(pl, p, st);
}

}  // namespace

extern "C" {

int mb_quantize(int32_t dtype, int64_t rows, int64_t cols, const void *x, int64_t ldx, int8_t *q, int64_t ldq,
                float *scale, void *stream) {
  if (!is_float(dtype)) return by_float(dtype, [](auto *) { return MB_OK; });
  int rc = check_rows(dtype, rows, cols, ldx, x, "quantize: x");
  if (!rc) rc = check_rows(MB_I8, rows, cols, ldq, q, "quantize: q");
  if (rc) return rc;
  if (rows == 0) return MB_OK;
  if (!scale) return fail(MB_ERR_INVALID, "quantize: null scale");
  if (rows > 0x7fff0000ll) return fail(MB_ERR_INVALID, "quantize: more than 2^31 - 2^16 rows");
  return by_float(dtype, [&](auto *tag) {
    using T = std::remove_pointer_t<decltype(tag)>;
    RouteParams p{};
    p.T = (int)rows; p.H = (int)cols; p.k = 1;
    p.src = x; p.ld_src = ldx; p.dst = q; p.ld_dst = ldq; p.scale = scale;
    return launch_quantize<T>(p, (cudaStream_t)stream, "quantize");
  });
}

void mb_scaled_desc_init(mb_scaled_desc *d) {
  if (d) memset(d, 0, sizeof(*d));
}

int64_t mb_scaled_workspace_size(const mb_scaled_desc *d) {
  SgPlan pl;
  if (scaled_check(d) || sg_plan(d, pl)) return 0;
  return pl.ws_bytes;
}

int mb_scaled_plan(const mb_scaled_desc *d, char *buf, int buflen) {
  SgPlan pl;
  int rc = scaled_check(d);
  if (!rc) rc = sg_plan(d, pl);
  if (rc) return -rc;
  const size_t room = buf ? (size_t)std::max(buflen, 0) : 0;
  if (pl.gemv) return snprintf(buf, room, "rows in one pass over the weights");
  if (pl.thin) return snprintf(buf, room, "rows in one pass over the weights, MMA, %d blocks an SM", pl.thin);
  if (pl.bn == 0) return snprintf(buf, room, pl.empty ? "empty" : "no sum");
  return snprintf(buf, room, "%s bn=%d pair=%d split=%d w_mn=%d pack_a=%d pack_b=%d ws=%lld",
                  pl.swap ? "channels" : "tokens", pl.bn, pl.pair, pl.split, pl.w_mn, pl.pk_a, pl.pk_b,
                  (long long)pl.ws_bytes);
}

int mb_scaled_gemm(const mb_scaled_desc *d, void *stream) {
  SgPlan pl;
  int rc = scaled_check(d);
  if (!rc) rc = sg_plan(d, pl);
  if (rc || pl.empty) return rc;
  if (pl.ws_bytes > 0 && (!d->workspace || d->workspace_bytes < pl.ws_bytes))
    return fail(MB_ERR_WORKSPACE, "workspace of %lld bytes required", (long long)pl.ws_bytes);
  if (pl.ws_bytes > 0 && !aligned16(d->workspace))  // operand copies are stored and loaded 16 bytes at a time
    return fail(MB_ERR_WORKSPACE, "the workspace must start on a 16-byte boundary");
  return by_float(d->out_dtype, [&](auto *tag) {
    return sg_launch<std::remove_pointer_t<decltype(tag)>>(d, pl, (cudaStream_t)stream);
  });
}

int mb_expert_sort(int32_t ids64, int64_t n, int64_t experts, const void *ids, int32_t *order, int32_t *position,
                   int32_t *offsets, void *stream) {
  if (n < 0 || n > 0x7fffffffll - 65536) return fail(MB_ERR_INVALID, "expert_sort: %lld entries", (long long)n);
  if (experts < 1 || experts > kMaxExperts)
    return fail(MB_ERR_INVALID, "expert_sort: %lld experts (1 to %d)", (long long)experts, kMaxExperts);
  if (!offsets || (n > 0 && (!ids || !order || !position))) return fail(MB_ERR_INVALID, "expert_sort: null pointer");
  SortParams p{ids, (int)n, (int)experts, order, position, offsets};
  int max_ranks = 0;
  const int rc = ids64 ? sort_setup<long long>(max_ranks) : sort_setup<int>(max_ranks);
  if (rc) return rc;
  // Blocks of few warps and many of them: a 32-warp block costs 2 us to start and
  // to step through its barriers, a cluster barrier 1 us, a warp's round of 32
  // entries 0.1 us, and the scattered stores of `order` bind an SM.  Up to 512
  // entries one block (4.1 us at 256 experts), then 256 entries a block up to 16
  // blocks, then 8 warps a block until a warp holds 256 entries.  Measured
  // against 1 to 16 blocks and 32 to 256 entries a warp: 1024 entries 4.5 us
  // (4.3 at best), 8192 5.2 (one block 14.7), 65536 10.9 (8 blocks 16.6).
  int ranks = 1;
  if (n > 512)
    while (ranks < max_ranks && n > (int64_t)ranks * 256) ranks *= 2;
  int64_t W = std::min<int64_t>(8, ceil_div(n, 64 * ranks));
  W = std::max(W, ceil_div(n, (int64_t)ranks * 32 * kSortBatch));  // the batch that lanes hold, while warps last
  W = std::min<int64_t>(32, std::max(W, ceil_div(experts, 32)));   // a thread per expert in the scan
  const int threads = (int)std::max<int64_t>(W, 1) * 32;
  const size_t smem = sort_smem(threads / 32, experts);
  auto kern = ids64 ? expert_sort_kernel<long long> : expert_sort_kernel<int>;
  return launch_pdl(kern, dim3(ranks), dim3(threads), smem, (cudaStream_t)stream, ranks, "expert_sort", p);
}

int mb_expert_gather(int32_t dtype, int64_t tokens, int64_t k, int64_t cols, const void *x, int64_t ldx,
                     const int32_t *position, const int32_t *kept, void *sorted, int64_t lds, void *stream) {
  if (!is_float(dtype)) return by_float(dtype, [](auto *) { return MB_OK; });
  int rc = check_route(tokens, k, cols, position, kept);
  if (!rc) rc = check_rows(dtype, tokens, cols, ldx, x, "expert_gather: x");
  if (!rc) rc = check_rows(dtype, tokens * k, cols, lds, sorted, "expert_gather: sorted");
  if (rc || tokens * k == 0 || cols == 0) return rc;
  return by_float(dtype, [&](auto *tag) {
    using T = std::remove_pointer_t<decltype(tag)>;
    RouteParams p{};
    p.T = (int)tokens; p.H = (int)cols; p.k = (int)k; p.position = position; p.kept = kept;
    p.src = x; p.ld_src = ldx; p.dst = sorted; p.ld_dst = lds;
    const bool al = rows16(x, ldx, sizeof(T)) && rows16(sorted, lds, sizeof(T)) && cols % Vec<T>::V == 0;
    const int lanes = route_lanes(cols, sizeof(T), false);
    auto kern = k <= 2 ? (al ? expert_gather_kernel<T, 2, true> : expert_gather_kernel<T, 2, false>)
                       : (al ? expert_gather_kernel<T, 4, true> : expert_gather_kernel<T, 4, false>);
    if constexpr (sizeof(T) == 2)
      if (k > 4 && al) kern = expert_gather_kernel<T, 8, true>;
    return launch_pdl(kern,
                      route_grid(tokens, cols, sizeof(T), lanes, false), dim3(kRouteThreads), 0, (cudaStream_t)stream, 1,
                      "expert_gather", p, lanes);
  });
}

int mb_expert_gather_quantize(int32_t dtype, int64_t tokens, int64_t k, int64_t cols, const void *x, int64_t ldx,
                              const int32_t *position, const int32_t *kept, int8_t *q, int64_t ldq, float *scale,
                              void *stream) {
  if (!is_float(dtype)) return by_float(dtype, [](auto *) { return MB_OK; });
  int rc = check_route(tokens, k, cols, position, kept);
  if (!rc) rc = check_rows(dtype, tokens, cols, ldx, x, "expert_gather_quantize: x");
  if (!rc) rc = check_rows(MB_I8, tokens * k, cols, ldq, q, "expert_gather_quantize: q");
  if (rc || tokens * k == 0) return rc;
  if (!scale) return fail(MB_ERR_INVALID, "expert_gather_quantize: null scale");
  return by_float(dtype, [&](auto *tag) {
    using T = std::remove_pointer_t<decltype(tag)>;
    RouteParams p{};
    p.T = (int)tokens; p.H = (int)cols; p.k = (int)k; p.position = position; p.kept = kept;
    p.src = x; p.ld_src = ldx; p.dst = q; p.ld_dst = ldq; p.scale = scale;
    return launch_quantize<T>(p, (cudaStream_t)stream, "expert_gather_quantize");
  });
}

int mb_expert_combine(int32_t dtype, int32_t weights_dtype, int64_t tokens, int64_t k, int64_t cols,
                      const void *sorted, int64_t lds, const void *weights, const int32_t *position,
                      const int32_t *kept, void *out, int64_t ldo, void *stream) {
  if (!is_float(dtype)) return by_float(dtype, [](auto *) { return MB_OK; });
  if (weights && weights_dtype != dtype && weights_dtype != MB_F32)
    return fail(MB_ERR_UNSUPPORTED, "expert_combine: weights must have the rows' type or fp32");
  int rc = check_route(tokens, k, cols, position, kept);
  if (!rc) rc = check_rows(dtype, tokens * k, cols, lds, sorted, "expert_combine: sorted");
  if (!rc) rc = check_rows(dtype, tokens, cols, ldo, out, "expert_combine: out");
  if (rc || tokens == 0 || cols == 0) return rc;
  return by_float(dtype, [&](auto *tag) {
    using T = std::remove_pointer_t<decltype(tag)>;
    RouteParams p{};
    p.T = (int)tokens; p.H = (int)cols; p.k = (int)k; p.position = position; p.kept = kept;
    p.src = sorted; p.ld_src = lds; p.w = weights; p.dst = out; p.ld_dst = ldo;
    const bool al = rows16(sorted, lds, sizeof(T)) && rows16(out, ldo, sizeof(T)) && cols % Vec<T>::V == 0;
    const int lanes = route_lanes(cols, sizeof(T), false);
    const bool f32 = weights_dtype == MB_F32;
    auto pick = [&](auto ne) {
      constexpr int NE = decltype(ne)::value;
      return al ? (f32 ? expert_combine_kernel<T, float, NE, true> : expert_combine_kernel<T, T, NE, true>)
                : (f32 ? expert_combine_kernel<T, float, NE, false> : expert_combine_kernel<T, T, NE, false>);
    };
    auto kern = k <= 2 ? pick(std::integral_constant<int, 2>()) : pick(std::integral_constant<int, 4>());
    if constexpr (sizeof(T) == 2)
      if (k > 4 && al) kern = f32 ? expert_combine_kernel<T, float, 8, true> : expert_combine_kernel<T, T, 8, true>;
    return launch_pdl(kern, route_grid(tokens, cols, sizeof(T), lanes, false), dim3(kRouteThreads), 0,
                      (cudaStream_t)stream, 1, "expert_combine", p, lanes);
  });
}

int mb_expert_combine_backward(int32_t dtype, int32_t weights_dtype, int64_t tokens, int64_t k, int64_t cols,
                               const void *dout, int64_t ldd, const void *sorted, int64_t lds, const void *weights,
                               const int32_t *position, const int32_t *kept, void *dsorted, int64_t ldds,
                               void *dweights, void *stream) {
  if (!is_float(dtype)) return by_float(dtype, [](auto *) { return MB_OK; });
  if (weights_dtype != dtype && weights_dtype != MB_F32)
    return fail(MB_ERR_UNSUPPORTED, "expert_combine_backward: weights must have the rows' type or fp32");
  int rc = check_route(tokens, k, cols, position, kept);
  if (!rc) rc = check_rows(dtype, tokens, cols, ldd, dout, "expert_combine_backward: dout");
  if (!rc) rc = check_rows(dtype, tokens * k, cols, lds, sorted, "expert_combine_backward: sorted");
  if (!rc) rc = check_rows(dtype, tokens * k, cols, ldds, dsorted, "expert_combine_backward: dsorted");
  if (rc || tokens * k == 0) return rc;
  if (!weights || !dweights) return fail(MB_ERR_INVALID, "expert_combine_backward: null weights or dweights");
  return by_float(dtype, [&](auto *tag) {
    using T = std::remove_pointer_t<decltype(tag)>;
    RouteParams p{};
    p.T = (int)tokens; p.H = (int)cols; p.k = (int)k; p.position = position; p.kept = kept;
    p.src = dout; p.ld_src = ldd; p.src2 = sorted; p.ld_src2 = lds; p.w = weights;
    p.dst = dsorted; p.ld_dst = ldds; p.dst2 = dweights;
    const bool al = rows16(dout, ldd, sizeof(T)) && rows16(sorted, lds, sizeof(T)) &&
                    rows16(dsorted, ldds, sizeof(T)) && cols % Vec<T>::V == 0;
    const int lanes = route_lanes(cols, sizeof(T), true);
    const bool f32 = weights_dtype == MB_F32;
    auto pick = [&](auto ne) {
      constexpr int NE = decltype(ne)::value;
      return al ? (f32 ? expert_combine_backward_kernel<T, float, NE, true> : expert_combine_backward_kernel<T, T, NE, true>)
                : (f32 ? expert_combine_backward_kernel<T, float, NE, false> : expert_combine_backward_kernel<T, T, NE, false>);
    };
    auto kern = k <= 2 ? pick(std::integral_constant<int, 2>()) : pick(std::integral_constant<int, 4>());
    return launch_pdl(kern, route_grid(tokens, cols, sizeof(T), lanes, true), dim3(kRouteThreads), 0,
                      (cudaStream_t)stream, 1, "expert_combine_backward", p, lanes);
  });
}

}  // extern "C"
