// Host fast path of the int8 and 4-bit products, the expert routing and the router,
// part of the torch C++ extension of fastpath.cpp.
//
// These operators are a few microseconds of GPU time in a decode step, less than
// checking their arguments and allocating their results costs in Python.  Each
// try_* function serves the plain call (CUDA tensors of the current device, the
// layouts a program normally has, no autograd) with the same checks, one call of
// the C ABI and the same results, and returns None for everything else, errors
// included: then the Python path runs, which resolves the layout, records the
// gradient or raises.
#pragma once
#include <torch/extension.h>
#include <c10/cuda/CUDAStream.h>

#include "../../include/metalblas_b200.h"

namespace fastops {

struct Ops {
  decltype(&mb_quantize) quantize = nullptr;
  decltype(&mb_scaled_gemm) scaled_gemm = nullptr;
  decltype(&mb_scaled_workspace_size) scaled_ws = nullptr;
  decltype(&mb_expert_sort) sort = nullptr;
  decltype(&mb_expert_gather) gather = nullptr;
  decltype(&mb_expert_gather_quantize) gather_quantize = nullptr;
  decltype(&mb_expert_combine) combine = nullptr;
  decltype(&mb_expert_combine_backward) combine_backward = nullptr;
  decltype(&mb_int4_quantize) int4_quantize = nullptr;
  decltype(&mb_int4_dequantize) int4_dequantize = nullptr;
  decltype(&mb_int4_gemm) int4_gemm = nullptr;
  decltype(&mb_int4_workspace_size) int4_ws = nullptr;
  decltype(&mb_expert_route) route = nullptr;
  decltype(&mb_expert_route_backward) route_backward = nullptr;
  decltype(&mb_expert_balance) balance = nullptr;
  decltype(&mb_expert_balance_workspace_size) balance_ws = nullptr;
  decltype(&mb_expert_balance_backward) balance_backward = nullptr;
};
inline Ops g_ops;

inline void set_ops(const std::vector<int64_t> &fn) {
  TORCH_CHECK(fn.size() == 17, "set_ops: 17 addresses expected");
  auto set = [&](auto &f, int i) { f = reinterpret_cast<std::remove_reference_t<decltype(f)>>(fn[i]); };
  set(g_ops.quantize, 0); set(g_ops.scaled_gemm, 1); set(g_ops.scaled_ws, 2); set(g_ops.sort, 3);
  set(g_ops.gather, 4); set(g_ops.gather_quantize, 5); set(g_ops.combine, 6); set(g_ops.combine_backward, 7);
  set(g_ops.int4_quantize, 8); set(g_ops.int4_dequantize, 9); set(g_ops.int4_gemm, 10); set(g_ops.int4_ws, 11);
  set(g_ops.route, 12); set(g_ops.route_backward, 13);
  set(g_ops.balance, 14); set(g_ops.balance_ws, 15); set(g_ops.balance_backward, 16);
}

// mb_dtype of a float tensor, or -1.
inline int float_code(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return MB_F32;
    case at::kHalf: return MB_F16;
    case at::kBFloat16: return MB_BF16;
    default: return -1;
  }
}
inline bool here(const at::Tensor &t, int dev) { return t.is_cuda() && t.get_device() == dev && !t.is_neg(); }
inline void *stream_of(int dev) { return reinterpret_cast<void *>(c10::cuda::getCurrentCUDAStream(dev).stream()); }
// A derivative to record or, with a tangent, to refuse: not a plain call.
inline bool grad_of(const at::Tensor &t) {
  return (t.requires_grad() && at::GradMode::is_enabled()) || t._fw_grad(/*level=*/0).defined();
}

// A matrix with contiguous, non-overlapping rows; its row stride.
inline bool rows_of(const at::Tensor &t, int dev, int64_t &ld) {
  if (t.dim() != 2 || !here(t, dev)) return false;
  const int64_t r = t.size(0), c = t.size(1);
  if (c > 1 && t.stride(1) != 1) return false;
  if (r > 1 && t.stride(0) < c) return false;
  ld = r > 1 ? t.stride(0) : c;
  return true;
}
inline at::Tensor int8_rows(int64_t rows, int64_t cols, const at::TensorOptions &o, int64_t &pitch) {
  pitch = (cols + 15) / 16 * 16;
  at::Tensor q = at::empty({rows, pitch}, o.dtype(at::kChar));
  return pitch == cols ? q : q.narrow(1, 0, cols);
}
// A contiguous tensor in the storage of a contiguous one.
inline at::Tensor part_of(const at::Tensor &all, int64_t offset, at::IntArrayRef sizes) {
  at::Tensor t = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(all.storage()), all.key_set(), all.dtype());
  t.unsafeGetTensorImpl()->set_storage_offset(offset);
  t.unsafeGetTensorImpl()->set_sizes_contiguous(sizes);
  return t;
}
inline at::TensorOptions plain_options(int dev, at::ScalarType t) {
  return at::TensorOptions().device(at::kCUDA, (c10::DeviceIndex)dev).dtype(t);
}

// position [T, k] and offsets [E + 1] as expert_sort makes them.
struct Order {
  int64_t T, k;
  const int32_t *position, *kept;
};
inline bool order_of(const at::Tensor &pos, const at::Tensor &off, int dev, Order &o) {
  if (!here(pos, dev) || !here(off, dev) || pos.scalar_type() != at::kInt || off.scalar_type() != at::kInt) return false;
  if (pos.dim() != 2 || off.dim() != 1 || off.size(0) < 2 || !pos.is_contiguous() || !off.is_contiguous()) return false;
  o.T = pos.size(0);
  o.k = pos.size(1);
  o.position = pos.data_ptr<int32_t>();
  o.kept = off.data_ptr<int32_t>() + off.size(0) - 1;
  return true;
}

using Pair = c10::optional<std::tuple<at::Tensor, at::Tensor>>;
using Triple = c10::optional<std::tuple<at::Tensor, at::Tensor, at::Tensor>>;
using One = c10::optional<at::Tensor>;

inline Pair try_quantize(const at::Tensor &x) {
  if (!g_ops.quantize || !x.is_cuda()) return c10::nullopt;
  const int dev = c10::cuda::current_device();
  int64_t ld, pitch;
  const int code = float_code(x.scalar_type());
  if (code < 0 || !rows_of(x, dev, ld)) return c10::nullopt;
  const int64_t rows = x.size(0), cols = x.size(1);
  at::Tensor q = int8_rows(rows, cols, plain_options(dev, at::kChar), pitch);
  at::Tensor scale = at::empty({rows}, plain_options(dev, at::kFloat));
  if (g_ops.quantize(code, rows, cols, x.data_ptr(), ld, (int8_t *)q.data_ptr(), pitch, scale.data_ptr<float>(),
                     stream_of(dev)) != MB_OK)
    return c10::nullopt;
  return std::make_tuple(q, scale);
}

// a [M, K], b [K, N] (E == 0) or [E, K, N] with offsets [E + 1].
inline One try_scaled(const at::Tensor &a, const at::Tensor &b, const at::Tensor &sa, const at::Tensor &sb,
                      const c10::optional<at::Tensor> &offsets, const c10::optional<at::Tensor> &bias,
                      at::ScalarType out_type) {
  if (!g_ops.scaled_gemm || !a.is_cuda()) return c10::nullopt;
  const int dev = c10::cuda::current_device();
  const int code = float_code(out_type), g = offsets.has_value() ? 1 : 0;
  if (code < 0 || a.dim() != 2 || b.dim() != 2 + g || sa.dim() != 1 || sb.dim() != 1 + g) return c10::nullopt;
  if (!here(a, dev) || !here(b, dev) || !here(sa, dev) || !here(sb, dev)) return c10::nullopt;
  if (a.scalar_type() != at::kChar || b.scalar_type() != at::kChar || sa.scalar_type() != at::kFloat ||
      sb.scalar_type() != at::kFloat)
    return c10::nullopt;
  const int64_t M = a.size(0), K = a.size(1), N = b.size(1 + g), E = g ? b.size(0) : 0;
  if (b.size(g) != K || sa.size(0) != M || sb.size(g) != N) return c10::nullopt;
  mb_scaled_desc d;
  memset(&d, 0, sizeof(d));
  d.out_dtype = d.bias_dtype = code;
  d.M = M; d.N = N; d.K = K; d.groups = E;
  if (g) {
    if (E < 1 || sb.size(0) != E || !here(*offsets, dev) || offsets->scalar_type() != at::kInt || offsets->dim() != 1 ||
        offsets->size(0) != E + 1 || !offsets->is_contiguous())
      return c10::nullopt;
    d.offsets = offsets->data_ptr<int32_t>();
    d.sB = b.stride(0);
    d.scale_b_g = sb.stride(0);
  }
  if (bias.has_value()) {
    const int bc = float_code(bias->scalar_type());
    if (!here(*bias, dev) || bias->dim() != 1 || bias->size(0) != N || (bc != code && bc != MB_F32)) return c10::nullopt;
    d.bias = bias->data_ptr();
    d.bias_s = bias->stride(0);
    d.bias_dtype = bc;
  }
  at::Tensor c = at::empty({M, N}, plain_options(dev, out_type)), ws;
  d.A = (const int8_t *)a.data_ptr(); d.B = (const int8_t *)b.data_ptr(); d.C = c.data_ptr();
  d.a_rs = a.stride(0); d.a_cs = a.stride(1);
  d.b_rs = b.stride(g); d.b_cs = b.stride(1 + g);
  d.c_rs = N; d.c_cs = 1;
  d.scale_a = sa.data_ptr<float>(); d.scale_a_s = sa.stride(0);
  d.scale_b = sb.data_ptr<float>(); d.scale_b_s = sb.stride(g);
  const int64_t need = g_ops.scaled_ws(&d);
  if (need > 0) {
    ws = at::empty({need}, plain_options(dev, at::kByte));
    d.workspace = ws.data_ptr();
    d.workspace_bytes = need;
  }
  if (g_ops.scaled_gemm(&d, stream_of(dev)) != MB_OK) return c10::nullopt;
  return c;
}

inline Triple try_sort(const at::Tensor &ids, int64_t experts) {
  if (!g_ops.sort || !ids.is_cuda()) return c10::nullopt;
  const int dev = c10::cuda::current_device();
  if (!here(ids, dev) || ids.dim() != 2 || !ids.is_contiguous()) return c10::nullopt;
  if (experts < 1 || experts > 1024) return c10::nullopt;  // mb_expert_sort's limit, before the allocation
  const bool wide = ids.scalar_type() == at::kLong;
  if (!wide && ids.scalar_type() != at::kInt) return c10::nullopt;
  const int64_t n = ids.numel();
  const auto i32 = plain_options(dev, at::kInt);
  const at::Tensor all = at::empty({2 * n + experts + 1}, i32);  // one allocation: 2 us less of 6.4
  const at::Tensor order = part_of(all, 0, {n}), position = part_of(all, n, ids.sizes()),
                   offsets = part_of(all, 2 * n, {experts + 1});
  if (g_ops.sort(wide, n, experts, ids.data_ptr(), order.data_ptr<int32_t>(), position.data_ptr<int32_t>(),
                 offsets.data_ptr<int32_t>(), stream_of(dev)) != MB_OK)
    return c10::nullopt;
  return std::make_tuple(order, position, offsets);
}

inline One try_gather(const at::Tensor &x, const at::Tensor &pos, const at::Tensor &off) {
  if (!g_ops.gather || !x.is_cuda() || grad_of(x)) return c10::nullopt;
  const int dev = c10::cuda::current_device();
  int64_t ld;
  Order o;
  const int code = float_code(x.scalar_type());
  if (code < 0 || !rows_of(x, dev, ld) || !order_of(pos, off, dev, o) || x.size(0) != o.T) return c10::nullopt;
  const int64_t H = x.size(1);
  at::Tensor out = at::empty({o.T * o.k, H}, plain_options(dev, x.scalar_type()));
  if (g_ops.gather(code, o.T, o.k, H, x.data_ptr(), ld, o.position, o.kept, out.data_ptr(), H, stream_of(dev)) != MB_OK)
    return c10::nullopt;
  return out;
}

inline Pair try_gather_quantize(const at::Tensor &x, const at::Tensor &pos, const at::Tensor &off) {
  if (!g_ops.gather_quantize || !x.is_cuda()) return c10::nullopt;
  const int dev = c10::cuda::current_device();
  int64_t ld, pitch;
  Order o;
  const int code = float_code(x.scalar_type());
  if (code < 0 || !rows_of(x, dev, ld) || !order_of(pos, off, dev, o) || x.size(0) != o.T) return c10::nullopt;
  const int64_t H = x.size(1), n = o.T * o.k;
  at::Tensor q = int8_rows(n, H, plain_options(dev, at::kChar), pitch);
  at::Tensor scale = at::empty({n}, plain_options(dev, at::kFloat));
  if (g_ops.gather_quantize(code, o.T, o.k, H, x.data_ptr(), ld, o.position, o.kept, (int8_t *)q.data_ptr(), pitch,
                            scale.data_ptr<float>(), stream_of(dev)) != MB_OK)
    return c10::nullopt;
  return std::make_tuple(q, scale);
}

// Contiguous weights like pos, of the rows' type or fp32.
inline bool weights_of(const at::Tensor &w, const at::Tensor &pos, int dev, int code, int &wcode) {
  wcode = float_code(w.scalar_type());
  return (wcode == code || wcode == MB_F32) && here(w, dev) && w.sizes() == pos.sizes() && w.is_contiguous();
}

inline One try_combine(const at::Tensor &rows, const c10::optional<at::Tensor> &w, const at::Tensor &pos,
                       const at::Tensor &off) {
  if (!g_ops.combine || !rows.is_cuda() || grad_of(rows) || (w.has_value() && grad_of(*w))) return c10::nullopt;
  const int dev = c10::cuda::current_device();
  int64_t ld;
  Order o;
  const int code = float_code(rows.scalar_type());
  int wcode = code;
  if (code < 0 || !rows_of(rows, dev, ld) || !order_of(pos, off, dev, o) || rows.size(0) != o.T * o.k) return c10::nullopt;
  if (w.has_value() && !weights_of(*w, pos, dev, code, wcode)) return c10::nullopt;
  const int64_t H = rows.size(1);
  at::Tensor out = at::empty({o.T, H}, plain_options(dev, rows.scalar_type()));
  if (g_ops.combine(code, wcode, o.T, o.k, H, rows.data_ptr(), ld, w.has_value() ? w->data_ptr() : nullptr, o.position,
                    o.kept, out.data_ptr(), H, stream_of(dev)) != MB_OK)
    return c10::nullopt;
  return out;
}

inline Pair try_combine_backward(const at::Tensor &grad, const at::Tensor &rows, const at::Tensor &w,
                                 const at::Tensor &pos, const at::Tensor &off) {
  if (!g_ops.combine_backward || !grad.is_cuda()) return c10::nullopt;
  const int dev = c10::cuda::current_device();
  int64_t ldg, ld;
  Order o;
  const int code = float_code(rows.scalar_type());
  int wcode;
  if (code < 0 || grad.scalar_type() != rows.scalar_type() || !rows_of(grad, dev, ldg) || !rows_of(rows, dev, ld) ||
      !order_of(pos, off, dev, o) || !weights_of(w, pos, dev, code, wcode))
    return c10::nullopt;
  const int64_t H = grad.size(1);
  if (grad.size(0) != o.T || rows.size(0) != o.T * o.k || rows.size(1) != H) return c10::nullopt;
  at::Tensor drows = at::empty({o.T * o.k, H}, plain_options(dev, rows.scalar_type()));
  at::Tensor dw = at::empty({o.T, o.k}, plain_options(dev, w.scalar_type()));
  if (g_ops.combine_backward(code, wcode, o.T, o.k, H, grad.data_ptr(), ldg, rows.data_ptr(), ld, w.data_ptr(),
                             o.position, o.kept, drows.data_ptr(), H, dw.data_ptr(), stream_of(dev)) != MB_OK)
    return c10::nullopt;
  return std::make_tuple(drows, dw);
}

// ------------------------------------------------------------------ 4-bit weights
inline bool group_of(int64_t g) { return g == 32 || g == 64 || g == 128 || g == 256; }

inline Pair try_int4_quantize(const at::Tensor &w, int64_t group, at::ScalarType scale_type) {
  if (!g_ops.int4_quantize || !w.is_cuda() || !group_of(group)) return c10::nullopt;
  const int dev = c10::cuda::current_device();
  int64_t ld;
  const int code = float_code(w.scalar_type()), sc = float_code(scale_type);
  if (code < 0 || sc < 0 || !rows_of(w, dev, ld)) return c10::nullopt;
  const int64_t rows = w.size(0), cols = w.size(1), bytes = (cols + 1) / 2, pitch = (bytes + 15) / 16 * 16;
  at::Tensor q = at::empty({rows, pitch}, plain_options(dev, at::kByte));
  at::Tensor scale = at::empty({rows, (cols + group - 1) / group}, plain_options(dev, scale_type));
  if (g_ops.int4_quantize(code, sc, rows, cols, (int32_t)group, w.data_ptr(), ld, q.data_ptr<uint8_t>(), pitch,
                          scale.data_ptr(), scale.size(1), stream_of(dev)) != MB_OK)
    return c10::nullopt;
  return std::make_tuple(pitch == bytes ? q : q.narrow(1, 0, bytes), scale);
}

// Rows of packed weights, their scales and zero points: [rows, .] matrices with contiguous rows.
inline bool weight_of(const at::Tensor &q, const at::Tensor &scale, const c10::optional<at::Tensor> &zero, int64_t cols,
                      int64_t group, int dim, int dev) {
  if (q.dim() != dim || scale.dim() != dim || !here(q, dev) || !here(scale, dev) || q.scalar_type() != at::kByte) return false;
  const int64_t bytes = (cols + 1) / 2, groups = (cols + group - 1) / group;
  auto fits = [&](const at::Tensor &t, int64_t n) {
    if (t.size(dim - 1) != n || (n > 1 && t.stride(dim - 1) != 1)) return false;
    if (t.size(dim - 2) != q.size(dim - 2) || (dim == 3 && t.size(0) != q.size(0))) return false;
    return (t.size(dim - 2) <= 1 || t.stride(dim - 2) >= n) && (dim < 3 || t.stride(0) >= 0);
  };
  if (!fits(q, bytes) || !fits(scale, groups)) return false;
  return !zero.has_value() || (here(*zero, dev) && zero->dim() == dim && zero->scalar_type() == at::kByte && fits(*zero, groups));
}

inline One try_int4_dequantize(const at::Tensor &q, const at::Tensor &scale, const c10::optional<at::Tensor> &zero,
                               int64_t cols, int64_t group, at::ScalarType out_type) {
  if (!g_ops.int4_dequantize || !q.is_cuda() || !group_of(group) || cols < 0) return c10::nullopt;
  const int dev = c10::cuda::current_device();
  const int code = float_code(out_type), sc = float_code(scale.scalar_type());
  if (code < 0 || sc < 0 || !weight_of(q, scale, zero, cols, group, 2, dev)) return c10::nullopt;
  const int64_t rows = q.size(0);
  at::Tensor out = at::empty({rows, cols}, plain_options(dev, out_type));
  if (g_ops.int4_dequantize(code, sc, rows, cols, (int32_t)group, q.data_ptr<uint8_t>(), q.stride(0), scale.data_ptr(),
                            scale.stride(0), zero.has_value() ? zero->data_ptr<uint8_t>() : nullptr,
                            zero.has_value() ? zero->stride(0) : 0, out.data_ptr(), cols, stream_of(dev)) != MB_OK)
    return c10::nullopt;
  return out;
}

// x [M, K]; weights [N, .], or [E, N, .] with offsets [E + 1].
inline One try_int4(const at::Tensor &x, const at::Tensor &q, const at::Tensor &scale, const c10::optional<at::Tensor> &zero,
                    int64_t group, const c10::optional<at::Tensor> &offsets, const c10::optional<at::Tensor> &bias) {
  if (!g_ops.int4_gemm || !x.is_cuda() || grad_of(x) || grad_of(scale) || (bias.has_value() && grad_of(*bias)) || !group_of(group))
    return c10::nullopt;
  const int dev = c10::cuda::current_device(), g = offsets.has_value() ? 1 : 0;
  int64_t ld;
  const at::ScalarType type = x.scalar_type();
  if ((type != at::kHalf && type != at::kBFloat16) || !rows_of(x, dev, ld)) return c10::nullopt;
  const int64_t M = x.size(0), K = x.size(1);
  if (!weight_of(q, scale, zero, K, group, 2 + g, dev) || (scale.scalar_type() != type && scale.scalar_type() != at::kFloat))
    return c10::nullopt;
  mb_int4_desc d;
  memset(&d, 0, sizeof(d));
  d.dtype = d.bias_dtype = float_code(type);
  d.scale_dtype = float_code(scale.scalar_type());
  d.group = (int32_t)group;
  d.M = M; d.N = q.size(g); d.K = K;
  d.x = x.data_ptr(); d.x_rs = ld;
  d.w = q.data_ptr<uint8_t>(); d.w_rs = q.stride(g);
  d.scale = scale.data_ptr(); d.scale_rs = scale.stride(g);
  if (zero.has_value()) {
    d.zero = zero->data_ptr<uint8_t>();
    d.zero_rs = zero->stride(g);
  }
  if (g) {
    const int64_t E = q.size(0);
    if (E < 1 || !here(*offsets, dev) || offsets->scalar_type() != at::kInt || offsets->dim() != 1 ||
        offsets->size(0) != E + 1 || !offsets->is_contiguous())
      return c10::nullopt;
    d.groups = E;
    d.offsets = offsets->data_ptr<int32_t>();
    d.w_e = q.stride(0);
    d.scale_e = scale.stride(0);
    if (zero.has_value()) d.zero_e = zero->stride(0);
  }
  if (bias.has_value()) {
    if (!here(*bias, dev) || bias->dim() != 1 || bias->size(0) != d.N || (d.N > 1 && bias->stride(0) != 1) ||
        (bias->scalar_type() != type && bias->scalar_type() != at::kFloat))
      return c10::nullopt;
    d.bias = bias->data_ptr();
    d.bias_dtype = float_code(bias->scalar_type());
  }
  at::Tensor out = at::empty({M, d.N}, plain_options(dev, type)), ws;
  d.out = out.data_ptr();
  d.out_rs = d.N;
  const int64_t need = g_ops.int4_ws(&d);
  if (need > 0) {
    ws = at::empty({need}, plain_options(dev, at::kByte));
    d.workspace = ws.data_ptr();
    d.workspace_bytes = need;
  }
  if (g_ops.int4_gemm(&d, stream_of(dev)) != MB_OK) return c10::nullopt;
  return out;
}

// ------------------------------------------------------------------ router
// Scores [T, E] of a float type; their row stride.
inline bool scores_of(const at::Tensor &x, int dev, int &code, int64_t &ld) {
  code = float_code(x.scalar_type());
  return code >= 0 && rows_of(x, dev, ld) && x.size(1) >= 1 && x.size(1) <= 1024;
}
// int32 expert numbers [T, k].
inline bool ids_of(const at::Tensor &ids, const at::Tensor &x, int dev) {
  return here(ids, dev) && ids.scalar_type() == at::kInt && ids.dim() == 2 && ids.size(0) == x.size(0) && ids.is_contiguous();
}
inline bool mask_of(const c10::optional<at::Tensor> &mask, const at::Tensor &x, int dev, const uint8_t *&p) {
  p = nullptr;
  if (!mask.has_value()) return true;
  if (!here(*mask, dev) || mask->scalar_type() != at::kBool || mask->dim() != 1 || mask->size(0) != x.size(0) || !mask->is_contiguous())
    return false;
  p = static_cast<const uint8_t *>(mask->data_ptr());
  return true;
}

inline Pair try_route(const at::Tensor &x, int64_t k, bool normalize) {
  if (!g_ops.route || !x.is_cuda() || grad_of(x)) return c10::nullopt;
  const int dev = c10::cuda::current_device();
  int code;
  int64_t ld;
  if (!scores_of(x, dev, code, ld) || k < 1 || k > x.size(1) || k > 64) return c10::nullopt;
  const int64_t T = x.size(0);
  at::Tensor w = at::empty({T, k}, plain_options(dev, at::kFloat)), ids = at::empty({T, k}, plain_options(dev, at::kInt));
  if (g_ops.route(code, T, x.size(1), k, normalize, x.data_ptr(), ld, w.data_ptr<float>(), ids.data_ptr<int32_t>(),
                  stream_of(dev)) != MB_OK)
    return c10::nullopt;
  return std::make_tuple(w, ids);
}

inline One try_route_backward(const at::Tensor &x, const at::Tensor &grad, const at::Tensor &ids, bool normalize) {
  if (!g_ops.route_backward || !x.is_cuda()) return c10::nullopt;
  const int dev = c10::cuda::current_device();
  int code;
  int64_t ld;
  if (!scores_of(x, dev, code, ld) || !ids_of(ids, x, dev)) return c10::nullopt;
  if (!here(grad, dev) || grad.scalar_type() != at::kFloat || grad.sizes() != ids.sizes() || !grad.is_contiguous()) return c10::nullopt;
  at::Tensor out = at::empty({x.size(0), x.size(1)}, plain_options(dev, x.scalar_type()));
  if (g_ops.route_backward(code, x.size(0), x.size(1), ids.size(1), normalize, grad.data_ptr<float>(), x.data_ptr(), ld,
                           ids.data_ptr<int32_t>(), out.data_ptr(), stream_of(dev)) != MB_OK)
    return c10::nullopt;
  return out;
}

inline Triple try_balance(const at::Tensor &x, const at::Tensor &ids, const c10::optional<at::Tensor> &mask) {
  if (!g_ops.balance || !x.is_cuda() || grad_of(x)) return c10::nullopt;
  const int dev = c10::cuda::current_device();
  int code;
  int64_t ld;
  const uint8_t *m;
  if (!scores_of(x, dev, code, ld) || !ids_of(ids, x, dev) || !mask_of(mask, x, dev, m)) return c10::nullopt;
  const int64_t T = x.size(0), E = x.size(1), need = g_ops.balance_ws(T, E);
  at::Tensor loss = at::empty({}, plain_options(dev, at::kFloat)), counts = at::empty({E}, plain_options(dev, at::kInt)),
             tokens = at::empty({}, plain_options(dev, at::kInt)), ws = at::empty({need}, plain_options(dev, at::kByte));
  if (g_ops.balance(code, T, E, ids.size(1), x.data_ptr(), ld, ids.data_ptr<int32_t>(), m, loss.data_ptr<float>(),
                    counts.data_ptr<int32_t>(), tokens.data_ptr<int32_t>(), ws.data_ptr(), need, stream_of(dev)) != MB_OK)
    return c10::nullopt;
  return std::make_tuple(loss, counts, tokens);
}

inline One try_balance_backward(const at::Tensor &x, const at::Tensor &grad, const at::Tensor &counts,
                                const at::Tensor &tokens, const c10::optional<at::Tensor> &mask) {
  if (!g_ops.balance_backward || !x.is_cuda()) return c10::nullopt;
  const int dev = c10::cuda::current_device();
  int code;
  int64_t ld;
  const uint8_t *m;
  if (!scores_of(x, dev, code, ld) || !mask_of(mask, x, dev, m)) return c10::nullopt;
  if (!here(grad, dev) || grad.scalar_type() != at::kFloat || grad.dim() != 0 || !here(counts, dev) ||
      counts.scalar_type() != at::kInt || counts.dim() != 1 || counts.size(0) != x.size(1) || !counts.is_contiguous() ||
      !here(tokens, dev) || tokens.scalar_type() != at::kInt || tokens.dim() != 0)
    return c10::nullopt;
  at::Tensor out = at::empty({x.size(0), x.size(1)}, plain_options(dev, x.scalar_type()));
  if (g_ops.balance_backward(code, x.size(0), x.size(1), grad.data_ptr<float>(), x.data_ptr(), ld, counts.data_ptr<int32_t>(),
                             tokens.data_ptr<int32_t>(), m, out.data_ptr(), stream_of(dev)) != MB_OK)
    return c10::nullopt;
  return out;
}

inline void bind(pybind11::module &m) {
  m.def("set_ops", &set_ops);
  // Arguments of other kinds (a scale that is no tensor) take the second form of
  // each name, so that the Python path's checks refuse them.
  auto def = [&](const char *name, auto fn) {
    m.def(name, fn);
    m.def(name, [](const pybind11::args &) { return pybind11::none(); });
  };
  def("try_quantize", &try_quantize);
  def("try_scaled", &try_scaled);
  def("try_sort", &try_sort);
  def("try_gather", &try_gather);
  def("try_gather_quantize", &try_gather_quantize);
  def("try_combine", &try_combine);
  def("try_combine_backward", &try_combine_backward);
  def("try_int4_quantize", &try_int4_quantize);
  def("try_int4_dequantize", &try_int4_dequantize);
  def("try_int4", &try_int4);
  def("try_route", &try_route);
  def("try_route_backward", &try_route_backward);
  def("try_balance", &try_balance);
  def("try_balance_backward", &try_balance_backward);
}

}  // namespace fastops
