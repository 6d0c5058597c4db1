"""Tokens sorted by expert and back, with gradients.

A mixture-of-experts layer sends each token to k of E experts.  ``expert_sort`` orders the
``T * k`` entries by expert on the device, ``expert_gather`` copies the tokens' rows into that
order (``expert_gather_quantize``: as int8 rows with scales), the experts' products run on
contiguous rows (``grouped_scaled_mm``), and ``expert_combine`` sums each token's k rows with
the router's weights.  Nothing here reads a count back to the host.

    order = expert_sort(ids, E)
    q, s = expert_gather_quantize(x, order)
    y = grouped_scaled_mm(q, w, s, sw, order.offsets)
    out = expert_combine(y, weights, order)

``expert_gather`` and ``expert_combine`` take part in reverse-mode autograd, once: a tangent
(forward mode) raises NotImplementedError, and so does differentiating their gradients again
(RuntimeError).  ``expert_gather_backward`` and ``expert_combine_backward`` are the gradients by
themselves; what they and ``expert_gather_quantize`` return carries no gradient.
"""
from __future__ import annotations

from typing import NamedTuple

import torch
import torch.autograd.forward_ad as fwd

from . import _lib
from .dispatch import FLOATS, _plain, _stream_of
from .quantized import _int8_rows, _ld, _on_device, _rows

MAX_EXPERTS = 1024

# The host fast path (csrc/fastops.h): the result of a plain call, or None.
_try_sort = _lib.fast_op("try_sort")
_try_gather = _lib.fast_op("try_gather")
_try_gather_quantize = _lib.fast_op("try_gather_quantize")
_try_combine = _lib.fast_op("try_combine")
_try_combine_backward = _lib.fast_op("try_combine_backward")


class ExpertOrder(NamedTuple):
    """The order of T tokens' entries by expert (int32 device tensors).

    order     [T * k]  entry ``t * k + j`` at each slot
    position  [T, k]   slot of each entry
    offsets   [E + 1]  first slot of each expert; ``offsets[E]`` is the number of entries
                       kept, and the slots from there on hold the dropped ones
    """
    order: torch.Tensor
    position: torch.Tensor
    offsets: torch.Tensor


def expert_sort(experts, num_experts):
    """``ExpertOrder`` of ``experts [T, k]`` (int32 or int64): entries by expert, those of one
    expert in their own order; numbers outside ``0 .. num_experts-1`` mark dropped entries."""
    fast = _try_sort(experts, num_experts)
    return ExpertOrder(*fast) if fast is not None else _sort(experts, num_experts)


@_on_device
def _sort(experts, num_experts):
    if experts.dtype not in (torch.int32, torch.int64):
        raise NotImplementedError(f"expert numbers must be int32 or int64, got {experts.dtype}")
    assert experts.dim() == 2, f"experts must be [tokens, k], got {tuple(experts.shape)}"
    if not 1 <= num_experts <= MAX_EXPERTS:
        raise ValueError(f"{num_experts} experts: 1 to {MAX_EXPERTS} expected")
    ids = experts.contiguous()
    n, dev = ids.numel(), ids.device
    order = torch.empty(n, dtype=torch.int32, device=dev)
    position = torch.empty(ids.shape, dtype=torch.int32, device=dev)
    offsets = torch.empty(num_experts + 1, dtype=torch.int32, device=dev)
    _lib.raise_for(_lib.load().mb_expert_sort(int(ids.dtype is torch.int64), n, num_experts, ids.data_ptr(),
                                              order.data_ptr(), position.data_ptr(), offsets.data_ptr(),
                                              _stream_of(dev)), "mb_expert_sort")
    return ExpertOrder(order, position, offsets)


def _check_order(order, dev):
    pos, off = order.position, order.offsets
    if pos.dtype is not torch.int32 or off.dtype is not torch.int32:
        raise NotImplementedError("ExpertOrder holds int32 tensors")
    assert pos.dim() == 2 and off.dim() == 1 and off.numel() >= 2, "position must be [T, k] and offsets [E + 1]"
    assert pos.device == dev and off.device == dev, "order and rows on different devices"
    return pos.contiguous(), off.contiguous()


def _check_rows(t, shape, name):
    assert isinstance(t, torch.Tensor), f"{name} must be a tensor"
    if t.dtype not in FLOATS:
        raise NotImplementedError(f"{name} must be fp32, fp16 or bf16, got {t.dtype}")
    assert tuple(t.shape) == tuple(shape), f"{name} has shape {tuple(t.shape)}, expected {tuple(shape)}"
    return _rows(t)


def _check_weights(weights, pos, dtype):
    assert isinstance(weights, torch.Tensor), "weights must be a tensor"
    assert weights.device == pos.device and tuple(weights.shape) == tuple(pos.shape), \
        f"weights have shape {tuple(weights.shape)}, expected {tuple(pos.shape)}"
    if weights.dtype is not dtype and weights.dtype is not torch.float32:
        raise NotImplementedError(f"weights must be {dtype} or fp32, got {weights.dtype}")
    return _plain(weights).contiguous()


def _kept(off):
    return off.data_ptr() + 4 * (off.numel() - 1)


@_on_device
def _gather(x, order):
    assert x.dim() == 2, f"x must be [T, cols], got {tuple(x.shape)}"
    pos, off = _check_order(order, x.device)
    T, k = pos.shape
    H = x.shape[1]
    x = _check_rows(x, (T, H), "x")
    out = torch.empty((T * k, H), dtype=x.dtype, device=x.device)
    _lib.raise_for(_lib.load().mb_expert_gather(_lib.DTYPE_CODE[x.dtype], T, k, H, x.data_ptr(), _ld(x),
                                                pos.data_ptr(), _kept(off), out.data_ptr(), H,
                                                _stream_of(x.device)), "mb_expert_gather")
    return out


@_on_device
def _combine(rows, weights, order):
    assert rows.dim() == 2, f"rows must be [T * k, cols], got {tuple(rows.shape)}"
    pos, off = _check_order(order, rows.device)
    T, k = pos.shape
    H = rows.shape[1]
    rows = _check_rows(rows, (T * k, H), "rows")
    pw, wd = None, rows.dtype
    if weights is not None:
        weights = _check_weights(weights, pos, rows.dtype)
        pw, wd = weights.data_ptr(), weights.dtype
    out = torch.empty((T, H), dtype=rows.dtype, device=rows.device)
    _lib.raise_for(_lib.load().mb_expert_combine(_lib.DTYPE_CODE[rows.dtype], _lib.DTYPE_CODE[wd], T, k, H,
                                                 rows.data_ptr(), _ld(rows), pw, pos.data_ptr(), _kept(off),
                                                 out.data_ptr(), H, _stream_of(rows.device)), "mb_expert_combine")
    return out


def _no_tangent(*tensors):
    for t in tensors:
        if isinstance(t, torch.Tensor) and fwd.unpack_dual(t).tangent is not None:
            raise NotImplementedError("expert_gather, expert_combine and their gradients have no forward-mode "
                                      "derivative")


class _Gather(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, order, position, offsets):
        ctx.save_for_backward(order, position, offsets)
        return _gather(x, ExpertOrder(order, position, offsets))

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        _no_tangent(grad)
        return expert_gather_backward(grad, ExpertOrder(*ctx.saved_tensors)), None, None, None


class _Combine(torch.autograd.Function):
    @staticmethod
    def forward(ctx, rows, weights, order, position, offsets):
        ctx.save_for_backward(rows, weights, order, position, offsets)
        return _combine(rows, weights, ExpertOrder(order, position, offsets))

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        rows, weights, *order = ctx.saved_tensors
        _no_tangent(grad)
        return (*expert_combine_backward(grad, rows, weights, ExpertOrder(*order)), None, None, None)


def expert_gather(x, order):
    """The rows of ``x [T, cols]`` in ``order``: ``[T * k, cols]``, zero rows for dropped entries.
    Takes part in reverse-mode autograd."""
    out = _try_gather(x, order.position, order.offsets)
    if out is not None:
        return out
    _no_tangent(x)
    if isinstance(x, torch.Tensor) and x.requires_grad and torch.is_grad_enabled():
        return _Gather.apply(x, *order)
    return _gather(x, order)


def expert_gather_backward(grad, order):
    """Gradient of ``expert_gather`` by x: each token's rows of ``grad [T * k, cols]`` summed.
    The result carries no gradient."""
    out = _try_combine(grad, None, order.position, order.offsets)
    return out if out is not None else _combine(grad, None, order)


def expert_gather_quantize(x, order):
    """``quantize(expert_gather(x, order))`` without the rows in between: int8 ``[T * k, cols]``
    and fp32 ``[T * k]``; dropped entries have q 0 and scale 0.  The result carries no gradient."""
    return _try_gather_quantize(x, order.position, order.offsets) or _gather_quantize(x, order)


@_on_device
def _gather_quantize(x, order):
    assert x.dim() == 2, f"x must be [T, cols], got {tuple(x.shape)}"
    pos, off = _check_order(order, x.device)
    T, k = pos.shape
    H = x.shape[1]
    x = _check_rows(x, (T, H), "x")
    q = _int8_rows(T * k, H, x.device)
    scale = torch.empty(T * k, dtype=torch.float32, device=x.device)
    _lib.raise_for(_lib.load().mb_expert_gather_quantize(_lib.DTYPE_CODE[x.dtype], T, k, H, x.data_ptr(), _ld(x),
                                                         pos.data_ptr(), _kept(off), q.data_ptr(),
                                                         max(q.stride(0), H), scale.data_ptr(),
                                                         _stream_of(x.device)), "mb_expert_gather_quantize")
    return q, scale


def expert_combine(rows, weights, order):
    """``out[t] = sum_j weights[t, j] * rows[position[t, j]]``: ``[T, cols]`` from the experts'
    ``rows [T * k, cols]``, dropped entries left out, summed in fp32 in the order of j.
    ``weights [T, k]`` have the rows' type or fp32; None stands for ones.  Takes part in
    reverse-mode autograd."""
    out = _try_combine(rows, weights, order.position, order.offsets)
    if out is not None:
        return out
    _no_tangent(rows, weights)
    if torch.is_grad_enabled() and any(isinstance(t, torch.Tensor) and t.requires_grad for t in (rows, weights)):
        if weights is None:
            weights = torch.ones(order.position.shape, dtype=torch.float32, device=rows.device)
        return _Combine.apply(rows, weights, *order)
    return _combine(rows, weights, order)


def expert_combine_backward(grad, rows, weights, order):
    """Gradients of ``expert_combine`` by rows and by weights: ``drows[position[t, j]] =
    weights[t, j] * grad[t]`` (zero for dropped entries) and ``dweights[t, j] = <grad[t],
    rows[position[t, j]]>`` (zero likewise), in the types of rows and weights.  The results carry
    no gradient."""
    return _try_combine_backward(grad, rows, weights, order.position, order.offsets) or \
        _combine_backward(grad, rows, weights, order)


@_on_device
def _combine_backward(grad, rows, weights, order):
    pos, off = _check_order(order, grad.device)
    T, k = pos.shape
    H = grad.shape[-1]
    assert isinstance(rows, torch.Tensor), "rows must be a tensor"
    if grad.dtype is not rows.dtype:
        raise NotImplementedError(f"grad is {grad.dtype}, rows are {rows.dtype}")
    assert rows.device == grad.device, "grad and rows on different devices"
    grad = _check_rows(grad, (T, H), "grad")
    rows = _check_rows(rows, (T * k, H), "rows")
    weights = _check_weights(weights, pos, rows.dtype)
    drows = torch.empty((T * k, H), dtype=rows.dtype, device=rows.device)
    dweights = torch.empty((T, k), dtype=weights.dtype, device=rows.device)
    _lib.raise_for(_lib.load().mb_expert_combine_backward(
        _lib.DTYPE_CODE[rows.dtype], _lib.DTYPE_CODE[weights.dtype], T, k, H, grad.data_ptr(), _ld(grad),
        rows.data_ptr(), _ld(rows), weights.data_ptr(), pos.data_ptr(), _kept(off), drows.data_ptr(), H,
        dweights.data_ptr(), _stream_of(rows.device)), "mb_expert_combine_backward")
    return drows, dweights
