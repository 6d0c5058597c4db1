// C ABI of the 4-bit weights (int4.cuh, int4_gemm.cuh).
#include <cuda.h>
#include <cuda_runtime.h>

#include <atomic>
#include <cmath>
#include <cstring>
#include <type_traits>

#include "mb_host.cuh"
#include "mb_common.cuh"
#include "int4.cuh"
#include "int4_gemm.cuh"
#include "int4_few.cuh"
#include "int4_tc.cuh"
#include "scaled_tc.cuh"

using namespace mb;
using namespace mb::host;

int mb::int4_status_read(int *v) {
  return cuda_check(cudaMemcpyFromSymbol(v, g_mb_status, sizeof(int)), "read status");
}
void mb::int4_status_clear() {
  int z = 0;
  cudaMemcpyToSymbol(g_mb_status, &z, sizeof(int));
}

namespace {

bool is_float(int dt) { return dt == MB_F32 || dt == MB_F16 || dt == MB_BF16; }
bool rows16(const void *p, int64_t rows, int64_t ld, int esz) { return aligned16(p) && (rows <= 1 || (ld * esz) % 16 == 0); }

int group_log2(int group) {
  switch (group) {
    case 32: return 5;
    case 64: return 6;
    case 128: return 7;
    case 256: return 8;
  }
  return 0;
}

// f(tag) with a null pointer of the element type.
template <class F>
int by_float(int dt, F &&f) {
  switch (dt) {
    case MB_F32: return f((float *)nullptr);
    case MB_F16: return f((__half *)nullptr);
    case MB_BF16: return f((__nv_bfloat16 *)nullptr);
  }
  return fail(MB_ERR_UNSUPPORTED, "dtype %d is not a float type (fp32, fp16, bf16)", dt);
}

int check_convert(const char *what, int dtype, int scale_dtype, int64_t rows, int64_t cols, int group, const void *x,
                  int64_t ldx, const uint8_t *q, int64_t ldq, const void *scale, int64_t lds) {
  if (!is_float(dtype) || !is_float(scale_dtype))
    return fail(MB_ERR_UNSUPPORTED, "%s: fp32, fp16 or bf16 expected, got %d and %d", what, dtype, scale_dtype);
  if (!group_log2(group)) return fail(MB_ERR_INVALID, "%s: a group has 32, 64, 128 or 256 columns, not %d", what, group);
  if (rows < 0 || cols < 0) return fail(MB_ERR_INVALID, "%s: negative extent", what);
  if (cols > (1ll << 30) || rows > (1ll << 40)) return fail(MB_ERR_INVALID, "%s: %lld x %lld", what, (long long)rows, (long long)cols);
  if (rows == 0 || cols == 0) return MB_OK;
  if (!x || !q || !scale) return fail(MB_ERR_INVALID, "%s: null pointer", what);
  if (rows > 1 && (ldx < cols || ldq < (cols + 1) / 2 || lds < ceil_div(cols, group)))
    return fail(MB_ERR_INVALID, "%s: rows overlap", what);
  return MB_OK;
}
// Spans of 256 columns that a warp of a conversion takes at a time, f(it, blocks): several where
// rows have them and there is work for every SM.
template <class F>
int by_spans(int64_t rows, int64_t cols, F &&f) {
  using std::integral_constant;
  const int64_t sms = device_sms(), most = sms * 32;
  auto blocks = [&](int b) { return (unsigned)std::min<int64_t>(ceil_div(rows * ceil_div(cols, 256 * b), 8), most); };
  if (cols > 512 && rows * ceil_div(cols, 1024) >= sms * 32) return f(integral_constant<int, 4>(), blocks(4));
  return f(integral_constant<int, 1>(), blocks(1));
}

int int4_check(const mb_int4_desc *d) {
  if (!d) return fail(MB_ERR_INVALID, "null descriptor");
  if (d->dtype != MB_F16 && d->dtype != MB_BF16) return fail(MB_ERR_UNSUPPORTED, "dtype %d is not fp16 or bf16", d->dtype);
  if (d->scale_dtype != d->dtype && d->scale_dtype != MB_F32)
    return fail(MB_ERR_UNSUPPORTED, "scales must have the tokens' type or fp32");
  if (!group_log2(d->group)) return fail(MB_ERR_INVALID, "a group has 32, 64, 128 or 256 columns, not %d", d->group);
  if (d->M < 0 || d->N < 0 || d->K < 0 || d->groups < 0) return fail(MB_ERR_INVALID, "negative extent");
  if (d->M > 0x7fff0000ll || d->N > 0x7fff0000ll || d->K > (1ll << 30))
    return fail(MB_ERR_INVALID, "M and N must stay below 2^31 - 2^16, K within 2^30");
  if (d->groups > i4::kMaxGroups) return fail(MB_ERR_INVALID, "more than %d groups", i4::kMaxGroups);
  if (d->M == 0 || d->N == 0) return MB_OK;
  if (!d->out) return fail(MB_ERR_INVALID, "null out");
  if (d->M > 1 && d->out_rs < d->N) return fail(MB_ERR_INVALID, "rows of out overlap");
  if (d->K > 0) {
    if (!d->x || !d->w || !d->scale) return fail(MB_ERR_INVALID, "null x, w or scale");
    if (d->M > 1 && d->x_rs < d->K) return fail(MB_ERR_INVALID, "rows of x overlap");
    if (d->N > 1 && d->w_rs < (d->K + 1) / 2) return fail(MB_ERR_INVALID, "rows of w overlap");
    if (d->w_rs < 0 || d->w_e < 0 || d->scale_rs < 0 || d->scale_e < 0 || d->zero_rs < 0 || d->zero_e < 0)
      return fail(MB_ERR_INVALID, "negative stride");
  }
  if (d->groups > 0 && !d->offsets) return fail(MB_ERR_INVALID, "groups need offsets");
  if (d->bias && d->bias_dtype != d->dtype && d->bias_dtype != MB_F32)
    return fail(MB_ERR_INVALID, "bias must have the tokens' type or fp32");
  return MB_OK;
}

// Rows of bytes that do not overlap one another.
struct ByteRows {
  uintptr_t at;
  int64_t rows, pitch, size;
  uintptr_t end() const { return at + (rows - 1) * pitch + size; }
};
bool share_bytes(ByteRows a, ByteRows b) {
  if (a.at > b.at) std::swap(a, b);
  if (b.at >= a.end()) return false;
  if (a.rows > 1 && b.rows > 1 && a.pitch == b.pitch) {   // b starts in a row of a, or in the space behind one
    const int64_t in = (int64_t)(b.at - a.at) % a.pitch;
    return in < a.size || in + b.size > a.pitch;
  }
  for (int64_t i = a.rows > 1 ? (int64_t)(b.at - a.at) / a.pitch : 0, j = 0; i < a.rows && j < b.rows;) {
    const uintptr_t p = a.at + i * a.pitch, q = b.at + j * b.pitch;
    if (p < q + b.size && q < p + a.size) return true;
    if (p < q) ++i;
    else ++j;
  }
  return false;
}
// Blocks write results while others still read.  (Of weights, scales and zero points all that lies
// between the first and the last counts.)
int check_out_apart(const mb_int4_desc *d) {
  auto at = [](const void *p) { return reinterpret_cast<uintptr_t>(p); };
  const ByteRows out{at(d->out), d->M, 2 * d->out_rs, 2 * d->N};
  const int64_t groups = ceil_div(d->K, d->group), last = d->groups > 1 ? d->groups - 1 : 0;
  auto meets = [&](const void *p, int64_t rs, int64_t e, int64_t n, int esz) {
    return p && d->K > 0 && share_bytes(out, ByteRows{at(p), 1, 0, (last * e + (d->N - 1) * rs + n) * esz});
  };
  const char *name = nullptr;
  if (d->K > 0 && share_bytes(out, ByteRows{at(d->x), d->M, 2 * d->x_rs, 2 * d->K})) name = "x";
  else if (meets(d->w, d->w_rs, d->w_e, (d->K + 1) / 2, 1)) name = "w";
  else if (meets(d->scale, d->scale_rs, d->scale_e, groups, elem_size(d->scale_dtype))) name = "scale";
  else if (meets(d->zero, d->zero_rs, d->zero_e, groups, 1)) name = "zero";
  else if (d->bias && share_bytes(out, ByteRows{at(d->bias), 1, 0, d->N * elem_size(d->bias_dtype)})) name = "bias";
  else if (d->groups && share_bytes(out, ByteRows{at(d->offsets), 1, 0, (d->groups + 1) * 4})) name = "offsets";
  return name ? fail(MB_ERR_INVALID, "out and %s share memory", name) : MB_OK;
}

i4::GemmArgs gemm_args(const mb_int4_desc *d) {
  i4::GemmArgs a{};
  a.x = d->x; a.x_rs = d->x_rs;
  a.M = (int)d->M; a.N = (int)d->N; a.K = (int)d->K; a.group_log2 = group_log2(d->group);
  a.w = d->w; a.w_rs = d->w_rs; a.w_e = d->w_e;
  a.scale = d->scale; a.s_rs = d->scale_rs; a.s_e = d->scale_e; a.scale_f32 = d->scale_dtype == MB_F32;
  a.zero = d->zero; a.z_rs = d->zero_rs; a.z_e = d->zero_e;
  a.bias = d->bias; a.bias_f32 = d->bias_dtype == MB_F32;
  a.groups = (int)d->groups; a.offsets = d->groups ? d->offsets : nullptr;
  a.out = d->out; a.out_rs = d->out_rs;
  return a;
}

template <class T, int LW, int NT, bool ZERO>
int few_launch_as(const i4::GemmArgs &a, cudaStream_t st) {
  constexpr auto kern = i4::int4_few_kernel<T, LW, NT, ZERO>;
  using Cfg = i4::FewCfg<NT>;
  int rc = allow_smem<kern>(Cfg::smem(i4::kMaxGroups));
  if (rc) return rc;
  CUtensorMap w{};
  const int64_t bytes = (a.K + 1) / 2;
  if (a.K > 0)   // boxes of 16 rows x 256 columns
    rc = encode_map(&w, MB_U8, a.w, bytes, a.N, a.w_e == 0 ? 1 : std::max(a.groups, 1), a.N == 1 ? round_up(bytes, 16) : a.w_rs, a.w_e,
                    i4::FEW_SLICE / 2, 16);
  if (rc) return rc;
  return launch_pdl(kern, dim3((unsigned)device_sms()), dim3(Cfg::THREADS), Cfg::smem(a.groups), st, 1, "int4_gemm", a, w,
                    wait_timeout_ns());
}
template <class T, int LW, int NT>
int few_launch_lw(const i4::GemmArgs &a, cudaStream_t st) {
  return a.zero ? few_launch_as<T, LW, NT, true>(a, st) : few_launch_as<T, LW, NT, false>(a, st);
}
template <class T, int NT>
int few_launch(const i4::GemmArgs &a, cudaStream_t st) {
  if (a.group_log2 == 5) return few_launch_lw<T, 1, NT>(a, st);
  return a.group_log2 == 6 ? few_launch_lw<T, 2, NT>(a, st) : few_launch_lw<T, 4, NT>(a, st);
}

template <class T, int BN, bool ZERO>
int tc_launch_as(i4::TcArgs &p, int split, int64_t units, cudaStream_t st) {
  constexpr auto kern = i4::int4_tc_kernel<T, BN, ZERO>;
  using Cfg = i4::TcCfg<BN>;
  const int rc = allow_smem<kern>(std::max(Cfg::smem(1, i4::kMaxGroups), Cfg::smem(Cfg::MAX_SPLIT, i4::kMaxGroups)));
  if (rc) return rc;
  p.split = split;
  const int64_t clusters = std::min<int64_t>(units, device_sms() / split);
  return launch_pdl(kern, dim3((unsigned)(clusters * split)), dim3(Cfg::THREADS), Cfg::smem(split, p.g.groups), st, split,
                    "int4_gemm", p);
}
template <class T, int BN>
int tc_launch_bn(i4::TcArgs &p, int split, int64_t units, cudaStream_t st) {
  return p.g.zero ? tc_launch_as<T, BN, true>(p, split, units, st) : tc_launch_as<T, BN, false>(p, split, units, st);
}

struct Plan {
  int few = 0;                 // tokens of a unit / 8 of the one-pass kernel, or 0
  int bn = 0, split = 1;       // tokens of a tile and CTAs that share it of the tcgen05 kernel
  int64_t units = 0;           // its units, at most
  int pk_x = 0, pk_w = 0;      // operand copied into the workspace first
  int64_t x_rs = 0, w_rs = 0, w_e = 0;
  int64_t x_off = 0, w_off = 0, ws_bytes = 0;
};

// Tiles of `rows` tokens that the groups are expected to have, groups of equal size at even odds.
// (They do not end on tiles' ends: half a tile more each.)
double expected_tiles(const mb_int4_desc *d, int rows) {
  if (!d->groups) return std::ceil((double)d->M / rows);
  const double E = (double)d->groups, used = E * (1.0 - std::pow(1.0 - 1.0 / E, (double)d->M)), each = d->M / used;
  return used * (each > rows / 2 ? each / rows + 0.5 : 1.0);
}
// A product's time in us by either kernel, fitted to times on B200.  The one-pass kernel: start,
// weights, and where units share blocks a second pass in most of them (a unit's slices of
// columns and tokens anew); passes of 112 rows; tokens.  Within 22 % over 160 dense products of
// 1 to 48 rows, K of 512 to 14336 and groups of 32 to 128 columns (7 % in the mean): 8 rows of 8192 x
// 2048 9.5 us, 9 rows 18.1 in two units of 8, 11.3 in one of 16.  The choice was the best of all forced
// plans or within 5 % of it in 69 of 73 products, 11 of them by group, 15 % over it at the worst.
double few_cost(const mb_int4_desc *d, int nt, int sms) {
  const double units = expected_tiles(d, 8 * nt), rows = units * d->N / sms, k = d->K * 1e-3;
  const double weight = (nt == 1 ? 0.169e-6 : 0.238e-6) * (d->group == 32 ? 1.36 : d->group == 64 ? 1.09 : 1.0);
  double t = (nt == 1 ? 4.7 + 0.1 * k : 5.2) + units * d->N * (double)d->K * weight;
  if (units > 1.0) t += nt == 1 ? 1.9 + 0.41 * k : 2.7 + 0.52 * k;
  return t + 2.8 * std::max(0.0, rows / 112 - 1.0) + 0.032 * std::min(d->M / units, 8.0 * nt) * k;
}
// The tcgen05 kernel: a step of 128 columns takes its MMA and decoding or, with several sums
// a step, the way of each accumulator to the sums and back.
double tc_cost(const mb_int4_desc *d, int bn, int split, int sms) {
  const double steps = std::ceil(d->K / 128.0) / split;
  const int sums = d->group < 128 ? 128 / d->group : 1;
  const double step = std::max(bn == 256 ? 1.02 : bn == 128 ? 0.62 : bn == 64 ? 0.57 : 0.52,
                               sums == 1 ? 0.0 : sums * (bn == 256 ? 0.65 : bn == 128 ? 0.4 : 0.36));
  const double tile = bn == 256 ? 3.0 : bn == 128 ? 1.5 : 1.0;
  // clusters of 4 and 8 leave SMs over in some GPCs
  const double slots = std::floor((double)sms / split * (split == 8 ? 0.75 : split == 4 ? 0.9 : 1.0));
  const double units = expected_tiles(d, bn) * (double)ceil_div(d->N, 128);
  const double waves = d->groups ? std::max(1.0, units / slots + 0.5) : std::ceil(units / slots);
  return 4.0 + waves * (tile + std::ceil(steps) * step) + 1.3 * std::log2((double)split);
}

int int4_plan(const mb_int4_desc *d, Plan &pl) {
  pl.x_rs = d->x_rs;
  pl.w_rs = d->w_rs;
  pl.w_e = d->w_e;
  if (d->M == 0 || d->N == 0) return MB_OK;
  const int64_t E = std::max<int64_t>(d->groups, 1), bytes = (d->K + 1) / 2;
  const int want = d->plan[0], split = d->plan[1], sms = device_sms();
  if (want != 0 && want != 1 && want != 2 && want != 16 && want != 32 && want != 64 && want != 128 && want != 256)
    return fail(MB_ERR_INVALID, "no plan %d", want);
  if (split != 0 && split != 1 && split != 2 && split != 4 && split != 8) return fail(MB_ERR_INVALID, "a split is 1, 2, 4 or 8");
  const int64_t stages = ceil_div(d->K, 256);
  double best = 1e300;
  for (const int nt : {1, 2}) {
    if (want ? want != nt || split > 1 : d->K > 0 && split) continue;
    // (the one-pass kernel counts rows of units in 32 bits)
    if ((ceil_div(d->M, 8 * nt) + (d->groups ? E : 0)) * d->N >= (1ll << 32)) continue;
    const double t = few_cost(d, nt, sms);
    if (t < best) {
      best = t;
      pl.few = nt;
    }
  }
  for (const int bn : {16, 32, 64, 128, 256}) {
    if (want ? want != bn : d->K == 0) continue;
    const int64_t units = (ceil_div(d->M, bn) + (d->groups ? std::min(E, d->M) : 0)) * ceil_div(d->N, 128);
    if (units >= (1ll << 31)) continue;
    for (const int sp : {1, 2, 4, 8}) {
      if (split ? split != sp : (units * sp > 2 * sms && sp > 1)) continue;
      if (sp > 1 && (bn == 256 || sp > stages)) continue;
      const double t = tc_cost(d, bn, sp, sms);
      if (t < best) {
        best = t;
        pl.few = 0;
        pl.bn = bn;
        pl.split = sp;
        pl.units = units;
      }
    }
  }
  if (!pl.few && !pl.bn) return fail(MB_ERR_INVALID, want || split ? "no kernel has plan %d with split %d" : "too many rows", want, split);
  int64_t at = 0;
  // tokens are read 16 bytes at a time; where their columns end inside these, only from rows that go on to
  // their end
  if (d->K > 0 && (!rows16(d->x, d->M, d->x_rs, 2) || (pl.few && d->K % 8))) {
    pl.pk_x = 1;
    pl.x_off = at;
    pl.x_rs = round_up(d->K, 8);
    at = round_up(at + d->M * pl.x_rs * 2, 256);
  }
  if (d->K > 0 && !(rows16(d->w, d->N, d->w_rs, 1) && (E == 1 || d->w_e % 16 == 0))) {
    pl.pk_w = 1;
    pl.w_off = at;
    pl.w_rs = round_up(bytes, 16);
    pl.w_e = d->w_e == 0 ? 0 : d->N * pl.w_rs;
    at = round_up(at + (d->w_e == 0 ? 1 : E) * d->N * pl.w_rs, 256);
  }
  pl.ws_bytes = at;
  return MB_OK;
}

template <class T>
int gemm_launch(const mb_int4_desc *d, const Plan &pl, cudaStream_t st) {
  i4::GemmArgs a = gemm_args(d);
  PackArgs px{}, pw{};
  const int64_t nw = d->w_e == 0 ? 1 : std::max<int64_t>(d->groups, 1);
  if (pl.pk_x) {   // rows as bytes
    px = PackArgs{d->x, static_cast<uint8_t *>(d->workspace) + pl.x_off, d->M, d->K * 2, d->x_rs * 2, 1, 0, 1, pl.x_rs * 2};
    a.x = px.dst;
    a.x_rs = pl.x_rs;
  }
  if (pl.pk_w) {
    pw = PackArgs{d->w, static_cast<uint8_t *>(d->workspace) + pl.w_off, d->N, (d->K + 1) / 2, d->w_rs, 1, d->w_e, nw, pl.w_rs};
    a.w = static_cast<uint8_t *>(pw.dst);
    a.w_rs = pl.w_rs;
    a.w_e = pl.w_e;
  }
  if (pl.pk_x || pl.pk_w) {
    auto blocks = [&](const PackArgs &m) {
      return m.dst ? std::min<int64_t>(ceil_div(m.batch * m.rows * ceil_div(m.cols, 512), 8), (int64_t)device_sms() * 4) : 0;
    };
    const int rc = launch_pdl(sg::scaled_pack_kernel, dim3((unsigned)(blocks(px) + blocks(pw))), dim3(256), 0, st, 1,
                              "int4_gemm: operand copy", px, pw, (int)blocks(px), d->w_e == 0 ? nullptr : a.offsets, a.M);
    if (rc) return rc;
  }
  if (pl.few) return pl.few == 2 ? few_launch<T, 2>(a, st) : few_launch<T, 1>(a, st);
  i4::TcArgs p{};
  p.g = a;
  p.tiles_n = (int)ceil_div(d->N, 128);
  p.steps = (int)ceil_div(d->K, i4::TC_STEP);
  p.out_vec = rows16(d->out, d->M, d->out_rs, 2);
  p.timeout_ns = wait_timeout_ns();
  const int64_t bytes = (d->K + 1) / 2;
  int rc = encode_map(&p.w, MB_U8, a.w, bytes, d->N, nw, d->N == 1 ? round_up(bytes, 16) : a.w_rs, a.w_e, 128, 128);
  if (!rc) rc = encode_map(&p.x, d->dtype, a.x, d->K, d->M, 1, d->M == 1 ? round_up(d->K, 8) : a.x_rs, 0, 64, std::min(pl.bn, 128));
  if (rc) return rc;
  switch (pl.bn) {
    case 16: return tc_launch_bn<T, 16>(p, pl.split, pl.units, st);
    case 32: return tc_launch_bn<T, 32>(p, pl.split, pl.units, st);
    case 64: return tc_launch_bn<T, 64>(p, pl.split, pl.units, st);
    case 128: return tc_launch_bn<T, 128>(p, pl.split, pl.units, st);
    default: return tc_launch_bn<T, 256>(p, pl.split, pl.units, st);
  }
}

}  // namespace

extern "C" {

int mb_int4_quantize(int32_t dtype, int32_t scale_dtype, int64_t rows, int64_t cols, int32_t group, const void *x,
                     int64_t ldx, uint8_t *q, int64_t ldq, void *scale, int64_t lds, void *stream) {
  const int rc = check_convert("int4_quantize", dtype, scale_dtype, rows, cols, group, x, ldx, q, ldq, scale, lds);
  if (rc || rows == 0 || cols == 0) return rc;
  i4::ConvertArgs a{x, ldx, q, ldq, rows, (int)cols, group_log2(group), scale, lds, nullptr, 0};
  return by_float(dtype, [&](auto *t) {
    return by_float(scale_dtype, [&](auto *s) {
      using T = std::remove_pointer_t<decltype(t)>;
      using S = std::remove_pointer_t<decltype(s)>;
      return by_spans(rows, cols, [&](auto b, unsigned blocks) {
        constexpr int B = decltype(b)::value;
        auto kern = rows16(x, rows, ldx, sizeof(T)) ? i4::quantize_int4_kernel<T, S, true, B> : i4::quantize_int4_kernel<T, S, false, B>;
        return launch_pdl(kern, dim3(blocks), dim3(256), 0, (cudaStream_t)stream, 1, "int4_quantize", a);
      });
    });
  });
}

int mb_int4_dequantize(int32_t dtype, int32_t scale_dtype, int64_t rows, int64_t cols, int32_t group, const uint8_t *q,
                       int64_t ldq, const void *scale, int64_t lds, const uint8_t *zero, int64_t ldz, void *out,
                       int64_t ldo, void *stream) {
  int rc = check_convert("int4_dequantize", dtype, scale_dtype, rows, cols, group, out, ldo, q, ldq, scale, lds);
  if (!rc && zero && rows > 1 && ldz < ceil_div(cols, group)) rc = fail(MB_ERR_INVALID, "int4_dequantize: rows overlap");
  if (rc || rows == 0 || cols == 0) return rc;
  i4::ConvertArgs a{q, ldq, out, ldo, rows, (int)cols, group_log2(group), const_cast<void *>(scale), lds, zero, ldz};
  return by_float(dtype, [&](auto *t) {
    return by_float(scale_dtype, [&](auto *s) {
      using T = std::remove_pointer_t<decltype(t)>;
      using S = std::remove_pointer_t<decltype(s)>;
      return by_spans(rows, cols, [&](auto b, unsigned blocks) {
        constexpr int B = decltype(b)::value;
        auto kern = rows16(out, rows, ldo, sizeof(T)) ? i4::dequantize_int4_kernel<T, S, true, B> : i4::dequantize_int4_kernel<T, S, false, B>;
        return launch_pdl(kern, dim3(blocks), dim3(256), 0, (cudaStream_t)stream, 1, "int4_dequantize", a);
      });
    });
  });
}

void mb_int4_desc_init(mb_int4_desc *d) {
  if (d) memset(d, 0, sizeof(*d));
}

int64_t mb_int4_workspace_size(const mb_int4_desc *d) {
  Plan pl;
  if (int4_check(d) || int4_plan(d, pl)) return 0;
  return pl.ws_bytes;
}

int mb_int4_plan(const mb_int4_desc *d, char *buf, int buflen) {
  Plan pl;
  int rc = int4_check(d);
  if (!rc) rc = int4_plan(d, pl);
  if (rc) return -rc;
  const size_t room = buf ? (size_t)std::max(buflen, 0) : 0;
  if (d->M == 0 || d->N == 0) return snprintf(buf, room, "empty");
  if (pl.few)
    return snprintf(buf, room, "units of %d tokens in one pass over the weights, pack_x=%d pack_w=%d ws=%lld", 8 * pl.few,
                    pl.pk_x, pl.pk_w, (long long)pl.ws_bytes);
  return snprintf(buf, room, "tiles of 128 rows x %d tokens, split=%d pack_x=%d pack_w=%d ws=%lld", pl.bn, pl.split, pl.pk_x,
                  pl.pk_w, (long long)pl.ws_bytes);
}

int mb_int4_gemm(const mb_int4_desc *d, void *stream) {
  Plan pl;
  int rc = int4_check(d);
  if (!rc) rc = int4_plan(d, pl);
  if (rc || d->M == 0 || d->N == 0) return rc;
  rc = check_out_apart(d);
  if (rc) return rc;
  if (pl.ws_bytes > 0 && (!d->workspace || d->workspace_bytes < pl.ws_bytes))
    return fail(MB_ERR_WORKSPACE, "workspace of %lld bytes required", (long long)pl.ws_bytes);
  if (pl.ws_bytes > 0 && !aligned16(d->workspace))  // operand copies are stored and loaded 16 bytes at a time
    return fail(MB_ERR_WORKSPACE, "the workspace must start on a 16-byte boundary");
  return d->dtype == MB_F16 ? gemm_launch<__half>(d, pl, (cudaStream_t)stream)
                            : gemm_launch<__nv_bfloat16>(d, pl, (cudaStream_t)stream);
}

}  // extern "C"
