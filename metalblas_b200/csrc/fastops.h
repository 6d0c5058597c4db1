// Host fast path of the int8 products with scales and the expert routing, part
// of the torch C++ extension of fastpath.cpp.
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
};
inline Ops g_ops;

inline void set_ops(const std::vector<int64_t> &fn) {
  TORCH_CHECK(fn.size() == 8, "set_ops: eight addresses expected");
  auto set = [&](auto &f, int i) { f = reinterpret_cast<std::remove_reference_t<decltype(f)>>(fn[i]); };
  set(g_ops.quantize, 0); set(g_ops.scaled_gemm, 1); set(g_ops.scaled_ws, 2); set(g_ops.sort, 3);
  set(g_ops.gather, 4); set(g_ops.gather_quantize, 5); set(g_ops.combine, 6); set(g_ops.combine_backward, 7);
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
}

}  // namespace fastops
