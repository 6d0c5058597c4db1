// C ABI of the 4-bit weights (int4.cuh, int4_gemm.cuh).
#include <cuda.h>
#include <cuda_runtime.h>

#include <atomic>
#include <cstring>
#include <type_traits>

#include "mb_host.cuh"
#include "mb_common.cuh"
#include "int4.cuh"
#include "int4_gemm.cuh"

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
unsigned convert_grid(int64_t rows, int64_t cols) {
  return (unsigned)std::min<int64_t>(ceil_div(rows * ceil_div(cols, 256), 8), (int64_t)device_sms() * 64);
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

template <class T>
int gemm_launch(const mb_int4_desc *d, cudaStream_t st) {
  const i4::GemmArgs a = gemm_args(d);
  const int64_t blocks = std::min<int64_t>(ceil_div(d->M * d->N, 8), (int64_t)device_sms() * 64);
  return launch_pdl(i4::int4_simple_kernel<T>, dim3((unsigned)blocks), dim3(256), 0, st, 1, "int4_gemm", a);
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
      auto kern = rows16(x, rows, ldx, sizeof(T)) ? i4::quantize_int4_kernel<T, S, true> : i4::quantize_int4_kernel<T, S, false>;
      return launch_pdl(kern, dim3(convert_grid(rows, cols)), dim3(256), 0, (cudaStream_t)stream, 1, "int4_quantize", a);
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
      auto kern = rows16(out, rows, ldo, sizeof(T)) ? i4::dequantize_int4_kernel<T, S, true> : i4::dequantize_int4_kernel<T, S, false>;
      return launch_pdl(kern, dim3(convert_grid(rows, cols)), dim3(256), 0, (cudaStream_t)stream, 1, "int4_dequantize", a);
    });
  });
}

void mb_int4_desc_init(mb_int4_desc *d) {
  if (d) memset(d, 0, sizeof(*d));
}

int64_t mb_int4_workspace_size(const mb_int4_desc *d) { return int4_check(d) ? 0 : 0; }

int mb_int4_plan(const mb_int4_desc *d, char *buf, int buflen) {
  const int rc = int4_check(d);
  if (rc) return -rc;
  return snprintf(buf, buf ? (size_t)std::max(buflen, 0) : 0, "simple");
}

int mb_int4_gemm(const mb_int4_desc *d, void *stream) {
  const int rc = int4_check(d);
  if (rc || d->M == 0 || d->N == 0) return rc;
  return d->dtype == MB_F16 ? gemm_launch<__half>(d, (cudaStream_t)stream) : gemm_launch<__nv_bfloat16>(d, (cudaStream_t)stream);
}

}  // extern "C"
