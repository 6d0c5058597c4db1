// C ABI of the int8 products with scales (quantize.cuh, scaled_gemm.cuh) and of
// the expert routing (experts.cuh).
#include <cuda.h>
#include <cuda_runtime.h>

#include <cstring>

#include "mb_host.cuh"
#include "mb_common.cuh"
#include "quantize.cuh"
#include "experts.cuh"
#include "scaled_gemm.cuh"

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
  if (rows > 1 && ld < cols) return fail(MB_ERR_INVALID, "%s: row stride %lld below %lld columns", what, (long long)ld, (long long)cols);
  if (rows > 0 && cols > 0 && !p) return fail(MB_ERR_INVALID, "%s: null pointer", what);
  return MB_OK;
}

int check_route(int64_t T, int64_t k, int64_t H, const int32_t *position, const int32_t *kept) {
  if (T < 0 || k < 0 || H < 0) return fail(MB_ERR_INVALID, "negative extent");
  if (k && T > 0x7fffffffll / k) return fail(MB_ERR_INVALID, "tokens * k must stay below 2^31");
  if (T * k > 0 && (!position || !kept)) return fail(MB_ERR_INVALID, "null position or kept");
  return MB_OK;
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
  if (rows > 0x7fffffff) return fail(MB_ERR_INVALID, "quantize: more than 2^31 - 1 rows");
  return by_float(dtype, [&](auto *tag) {
    using T = std::remove_pointer_t<decltype(tag)>;
    RouteParams p{};
    p.T = rows; p.H = cols; p.k = 1;
    p.src = x; p.ld_src = ldx; p.dst = q; p.ld_dst = ldq; p.scale = scale;
    constexpr int V = 16 / sizeof(T);
    const bool vec = rows16(x, ldx, sizeof(T)) && cols % V == 0;
    return launch_pdl(vec ? quantize_rows_kernel<T, V> : quantize_rows_kernel<T, 1>, dim3((unsigned)rows), dim3(256), 0,
                      (cudaStream_t)stream, 1, "quantize", p);
  });
}

void mb_scaled_desc_init(mb_scaled_desc *d) {
  if (d) memset(d, 0, sizeof(*d));
}

static int scaled_check(const mb_scaled_desc *d) {
  if (!d) return fail(MB_ERR_INVALID, "null descriptor");
  if (!is_float(d->out_dtype)) return fail(MB_ERR_UNSUPPORTED, "out_dtype %d is not fp32, fp16 or bf16", d->out_dtype);
  if (d->M < 0 || d->N < 0 || d->K < 0 || d->groups < 0) return fail(MB_ERR_INVALID, "negative extent");
  if (d->M > 0x7fffff00ll || d->N > 0x7fffff00ll) return fail(MB_ERR_INVALID, "M and N must stay below 2^31");
  if (d->K > 131071) return fail(MB_ERR_INVALID, "K = %lld: sums of more than 131071 int8 products can leave 32 bits", (long long)d->K);
  if (d->groups > 1024) return fail(MB_ERR_INVALID, "more than 1024 groups");
  if (d->M == 0 || d->N == 0) return MB_OK;
  if (!d->C || !d->scale_a || !d->scale_b) return fail(MB_ERR_INVALID, "null C, scale_a or scale_b");
  if (d->K > 0 && (!d->A || !d->B)) return fail(MB_ERR_INVALID, "null A or B");
  if (d->groups > 0 && !d->offsets) return fail(MB_ERR_INVALID, "groups need offsets");
  if (d->bias && d->bias_dtype != d->out_dtype && d->bias_dtype != MB_F32)
    return fail(MB_ERR_INVALID, "bias must have the output's type or fp32");
  return MB_OK;
}

int64_t mb_scaled_workspace_size(const mb_scaled_desc *d) { return 0; }

int mb_scaled_plan(const mb_scaled_desc *d, char *buf, int buflen) {
  const int rc = scaled_check(d);
  if (rc) return -rc;
  return snprintf(buf, buf ? (size_t)std::max(buflen, 0) : 0, "simple");
}

int mb_scaled_gemm(const mb_scaled_desc *d, void *stream) {
  const int rc = scaled_check(d);
  if (rc || d->M == 0 || d->N == 0) return rc;
  return by_float(d->out_dtype, [&](auto *tag) {
    using T = std::remove_pointer_t<decltype(tag)>;
    ScaledParams p{};
    p.M = d->M; p.N = d->N; p.K = d->K; p.groups = (int)std::max<int64_t>(d->groups, 1);
    p.A = d->A; p.B = d->B; p.C = d->C;
    p.a_rs = d->a_rs; p.a_cs = d->a_cs; p.b_rs = d->b_rs; p.b_cs = d->b_cs; p.sB = d->sB;
    p.c_rs = d->c_rs; p.c_cs = d->c_cs;
    p.scale_a = d->scale_a; p.scale_b = d->scale_b;
    p.sa_s = d->scale_a_s; p.sb_s = d->scale_b_s; p.sb_g = d->scale_b_g;
    p.bias = d->bias; p.bias_s = d->bias_s; p.bias_f32 = d->bias_dtype == MB_F32;
    p.offsets = d->groups ? d->offsets : nullptr;
    return launch_pdl(scaled_simple_kernel<T>, dim3((unsigned)(device_sms() * 8)), dim3(256), 0, (cudaStream_t)stream, 1,
                      "scaled_gemm", p);
  });
}

int mb_expert_sort(int32_t ids64, int64_t n, int64_t experts, const void *ids, int32_t *order, int32_t *position,
                   int32_t *offsets, void *stream) {
  if (n < 0 || n > 0x7fffffffll - 65536) return fail(MB_ERR_INVALID, "expert_sort: %lld entries", (long long)n);
  if (experts < 1 || experts > kMaxExperts)
    return fail(MB_ERR_INVALID, "expert_sort: %lld experts (1 to %d)", (long long)experts, kMaxExperts);
  if (!offsets || (n > 0 && (!ids || !order || !position))) return fail(MB_ERR_INVALID, "expert_sort: null pointer");
  SortParams p{ids, (int)n, (int)experts, order, position, offsets};
  const int W = (int)std::max<int64_t>(1, std::min<int64_t>(32, ceil_div(n, 32)));
  const size_t smem = (size_t)W * (experts + 1) * 4;
  auto kern = ids64 ? expert_sort_kernel<long long> : expert_sort_kernel<int>;
  const int rc = cuda_check(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem),
                            "cudaFuncSetAttribute");
  if (rc) return rc;
  return launch_pdl(kern, dim3(1), dim3(W * 32), smem, (cudaStream_t)stream, 1, "expert_sort", p);
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
    p.T = tokens; p.H = cols; p.k = (int)k; p.position = position; p.kept = kept;
    p.src = x; p.ld_src = ldx; p.dst = sorted; p.ld_dst = lds;
    constexpr int V = 16 / sizeof(T);
    const bool vec = rows16(x, ldx, sizeof(T)) && rows16(sorted, lds, sizeof(T)) && cols % V == 0;
    const dim3 grid((unsigned)tokens, (unsigned)std::min<int64_t>(ceil_div(cols, 256 * (vec ? V : 1)), 16));
    return launch_pdl(vec ? expert_gather_kernel<T, V> : expert_gather_kernel<T, 1>, grid, dim3(256), 0,
                      (cudaStream_t)stream, 1, "expert_gather", p);
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
    p.T = tokens; p.H = cols; p.k = (int)k; p.position = position; p.kept = kept;
    p.src = x; p.ld_src = ldx; p.dst = q; p.ld_dst = ldq; p.scale = scale;
    constexpr int V = 16 / sizeof(T);
    const bool vec = rows16(x, ldx, sizeof(T)) && cols % V == 0;
    return launch_pdl(vec ? quantize_rows_kernel<T, V> : quantize_rows_kernel<T, 1>, dim3((unsigned)tokens), dim3(256),
                      0, (cudaStream_t)stream, 1, "expert_gather_quantize", p);
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
    p.T = tokens; p.H = cols; p.k = (int)k; p.position = position; p.kept = kept;
    p.src = sorted; p.ld_src = lds; p.w = weights; p.dst = out; p.ld_dst = ldo;
    constexpr int V = 16 / sizeof(T);
    const bool vec = rows16(sorted, lds, sizeof(T)) && rows16(out, ldo, sizeof(T)) && cols % V == 0;
    const dim3 grid((unsigned)tokens, (unsigned)std::min<int64_t>(ceil_div(cols, 256 * (vec ? V : 1)), 16));
    const bool f32 = weights_dtype == MB_F32;
    auto kern = vec ? (f32 ? expert_combine_kernel<T, float, V> : expert_combine_kernel<T, T, V>)
                    : (f32 ? expert_combine_kernel<T, float, 1> : expert_combine_kernel<T, T, 1>);
    return launch_pdl(kern, grid, dim3(256), 0, (cudaStream_t)stream, 1, "expert_combine", p);
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
    p.T = tokens; p.H = cols; p.k = (int)k; p.position = position; p.kept = kept;
    p.src = dout; p.ld_src = ldd; p.src2 = sorted; p.ld_src2 = lds; p.w = weights;
    p.dst = dsorted; p.ld_dst = ldds; p.dst2 = dweights;
    constexpr int V = 16 / sizeof(T);
    const bool vec = rows16(dout, ldd, sizeof(T)) && rows16(sorted, lds, sizeof(T)) &&
                     rows16(dsorted, ldds, sizeof(T)) && cols % V == 0;
    const bool f32 = weights_dtype == MB_F32;
    auto kern = vec ? (f32 ? expert_combine_backward_kernel<T, float, V> : expert_combine_backward_kernel<T, T, V>)
                    : (f32 ? expert_combine_backward_kernel<T, float, 1> : expert_combine_backward_kernel<T, T, 1>);
    return launch_pdl(kern, dim3((unsigned)tokens), dim3(256), 0, (cudaStream_t)stream, 1, "expert_combine_backward",
                      p);
  });
}

}  // extern "C"
