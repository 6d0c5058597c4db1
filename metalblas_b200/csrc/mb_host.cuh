// Host helpers shared by the library's translation units (mb_abi.cu, mb_ops.cu):
// the thread's error text, status mapping, launches and tensor maps.
#pragma once
#include <cuda.h>
#include <cudaTypedefs.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdarg>
#include <cstdint>
#include <cstdio>
#include <cstdlib>
#include <mutex>
#include <string>
#include <utility>

#include "../../include/metalblas_b200.h"

namespace mb {
namespace host {

// Text of the last error on this thread (mb_last_error_string).
inline thread_local std::string g_err;

inline int fail(int code, const char *fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof(buf), fmt, ap);
  va_end(ap);
  g_err = buf;
  return code;
}

inline int cuda_check(cudaError_t e, const char *what) {
  if (e == cudaSuccess) return MB_OK;
  return fail(MB_ERR_LAUNCH, "%s: %s", what, cudaGetErrorString(e));
}

inline int elem_size(int dt) {
  switch (dt) {
    case MB_F32: return 4;
    case MB_F16: case MB_BF16: return 2;
    case MB_C64: return 8;
    case MB_C32: return 4;
    case MB_I8: case MB_U8: return 1;
    case MB_I16: return 2;
    case MB_I32: return 4;
    case MB_I64: return 8;
  }
  return 0;
}

inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
inline int64_t round_up(int64_t a, int64_t b) { return ceil_div(a, b) * b; }
inline bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// Limit of every device-side wait (METALBLAS_WAIT_TIMEOUT_MS, 2000 by default).
inline unsigned long long wait_timeout_ns() {
  static unsigned long long v = [] {
    const char *s = getenv("METALBLAS_WAIT_TIMEOUT_MS");
    long long ms = s ? atoll(s) : 2000;
    if (ms <= 0) ms = 2000;
    return (unsigned long long)ms * 1000000ull;
  }();
  return v;
}

// Programmatic dependent launch (see pdl_trigger / pdl_wait in mb_common.cuh);
// METALBLAS_PDL=0 launches with plain stream order.
inline bool pdl_enabled() {
  static const bool v = [] {
    const char *s = getenv("METALBLAS_PDL");
    return !(s && s[0] == '0');
  }();
  return v;
}

template <class... KArgs, class... Args>
int launch_pdl(void (*kern)(KArgs...), dim3 grid, dim3 block, size_t smem, cudaStream_t st, int cluster_x,
               const char *what, Args &&...args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  int n = 0;
  if (cluster_x > 1) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = cluster_x;
    attr[n].val.clusterDim.y = 1;
    attr[n].val.clusterDim.z = 1;
    ++n;
  }
  if (pdl_enabled()) {
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n].val.programmaticStreamSerializationAllowed = 1;
    ++n;
  }
  cfg.attrs = attr;
  cfg.numAttrs = n;
  return cuda_check(cudaLaunchKernelEx(&cfg, kern, std::forward<Args>(args)...), what);
}

inline PFN_cuTensorMapEncodeTiled_v12000 get_encode() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void *p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
  });
  return fn;
}

inline CUtensorMapDataType tma_dtype(int dt) {
  switch (dt) {
    case MB_BF16: return CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
    case MB_F16: return CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    case MB_F32: return CU_TENSOR_MAP_DATA_TYPE_FLOAT32;
    default: return CU_TENSOR_MAP_DATA_TYPE_UINT8;
  }
}

// 3-D tiled map {inner, outer, batch} with SWIZZLE_128B.
inline int encode_map(CUtensorMap *m, int dt, const void *base, int64_t inner, int64_t outer, int64_t batch,
                      int64_t outer_stride_el, int64_t batch_stride_el, int box_inner, int box_outer,
                      CUtensorMapSwizzle swz = CU_TENSOR_MAP_SWIZZLE_128B) {
  auto enc = get_encode();
  if (!enc) return fail(MB_ERR_LAUNCH, "cuTensorMapEncodeTiled unavailable");
  const int esz = elem_size(dt);
  cuuint64_t dims[3] = {(cuuint64_t)inner, (cuuint64_t)outer, (cuuint64_t)std::max<int64_t>(batch, 1)};
  int64_t ostr = outer_stride_el * esz;
  int64_t bstr = batch_stride_el * esz;
  if (batch <= 1 || bstr == 0) bstr = round_up(std::max<int64_t>(ostr * outer, 16), 16);
  cuuint64_t strides[2] = {(cuuint64_t)ostr, (cuuint64_t)bstr};
  cuuint32_t box[3] = {(cuuint32_t)box_inner, (cuuint32_t)box_outer, 1};
  cuuint32_t estr[3] = {1, 1, 1};
  CUresult r = enc(m, tma_dtype(dt), 3, const_cast<void *>(base), dims, strides, box, estr,
                   CU_TENSOR_MAP_INTERLEAVE_NONE, swz, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                   CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(MB_ERR_LAUNCH, "cuTensorMapEncodeTiled failed (%d)", (int)r);
  return MB_OK;
}

// SM count of the current device.
int device_sms();

}  // namespace host

// Device status word of the second translation unit (mb_ops.cu keeps its own,
// since each unit's kernels write the word of their module).
int ops_status_read(int *v);
void ops_status_clear();

}  // namespace mb
