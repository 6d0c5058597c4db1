"""Weights of 4 bits with group scales, and products of 16-bit tokens with them.

``quantize_int4`` packs a weight matrix two values to a byte with one scale for every group of
columns; ``int4_mm`` multiplies tokens with it and ``grouped_int4_mm`` does so with one weight
matrix per group of rows, as a mixture-of-experts layer has them after ``expert_sort``;
``dequantize_int4`` gives the weights back.

A weight is ``(u - zero) * scale`` with u in 0..15 and zero 8 unless zero points are given, so
weights of other tools (nibbles in the order of the columns, the even column low) are read as
they are.  The integers are exact in the tokens' type and the scales are applied to fp32 sums:
the weights are never rounded, whatever the number of rows.

The products have no gradient: 4-bit weights are constants of a serving program.  Tokens, scales,
biases and an ``out`` that require one are refused.
"""
from __future__ import annotations

import ctypes

import torch
import torch.autograd.forward_ad as fwd

from . import _lib
from .dispatch import FLOATS, _plain, _stream_of
from .quantized import MAX_GROUPS, _ld, _on_device, _rows

GROUP_SIZES = (32, 64, 128, 256)
TOKENS = (torch.float16, torch.bfloat16)

_byref = ctypes.byref
# The host fast path (csrc/fastops.h): the result of a plain call, or None.
_try_quantize = _lib.fast_op("try_int4_quantize")
_try_dequantize = _lib.fast_op("try_int4_dequantize")
_try_int4 = _lib.fast_op("try_int4")


def _group(group_size):
    if group_size not in GROUP_SIZES:
        raise ValueError(f"group_size must be 32, 64, 128 or 256, got {group_size}")
    return int(group_size)


def _groups(cols, group_size):
    return (cols + group_size - 1) // group_size


def _packed_rows(lead, cols, device):
    """uint8 rows of cols 4-bit values on 16-byte boundaries."""
    n = (cols + 1) // 2
    pitch = (n + 15) // 16 * 16
    q = torch.empty((*lead, pitch), dtype=torch.uint8, device=device)
    return q if pitch == n else q[..., :n]


def quantize_int4(w, group_size=128, *, scale_dtype=torch.float32):
    """Rows of ``w [..., cols]`` (fp32, fp16 or bf16) as ``(q, scale)``: uint8 ``q [..., (cols + 1)
    // 2]`` with two values to a byte, and ``scale [..., ceil(cols / group_size)]``.

    ``scale = max|w| / 7`` of a group in fp32, rounded to ``scale_dtype`` (fp32, fp16 or bf16; one
    that the type cannot hold is infinite), and ``u = 8 + round(w / scale)``, halves to even, so that
    ``w ~ (u - 8) * scale``.  A group of zeros has scale 0; one with an infinity or a NaN has
    scale NaN; both have u 8.  ``group_size`` is 32, 64, 128 or 256, the last group of a row may
    be shorter.  The rows of ``q`` start on 16-byte boundaries: with a number of columns that is
    no multiple of 32, ``q`` is a view of a wider tensor.  Neither carries a gradient.
    """
    return _try_quantize(w, group_size, scale_dtype) or _quantize(w, group_size, scale_dtype)


@_on_device
def _quantize(w, group_size, scale_dtype):
    G = _group(group_size)
    if w.dtype not in FLOATS or scale_dtype not in FLOATS:
        raise NotImplementedError(f"quantize_int4 takes fp32, fp16 or bf16, got {w.dtype} and {scale_dtype}")
    assert w.dim() >= 1, "quantize_int4 takes rows"
    lead, cols = w.shape[:-1], w.shape[-1]
    w2 = _rows(w if w.dim() == 2 else w.reshape(lead.numel(), cols))
    q = _packed_rows(lead, cols, w.device)
    scale = torch.empty((*lead, _groups(cols, G)), dtype=scale_dtype, device=w.device)
    rows = lead.numel()
    pitch = ((cols + 1) // 2 + 15) // 16 * 16
    _lib.raise_for(_lib.load().mb_int4_quantize(_lib.DTYPE_CODE[w.dtype], _lib.DTYPE_CODE[scale_dtype], rows, cols, G,
                                                w2.data_ptr(), _ld(w2), q.data_ptr(), pitch, scale.data_ptr(),
                                                scale.shape[-1], _stream_of(w.device)), "mb_int4_quantize")
    return q, scale


def _check_weight(q, scale, zero, cols, G, lead, dev):
    """Packed weights, scales and zero points of shape [*lead, .], their last dimension contiguous."""
    assert isinstance(q, torch.Tensor) and q.device == dev, f"weights must be a tensor on {dev}"
    if q.dtype is not torch.uint8:
        raise NotImplementedError(f"packed weights are uint8, got {q.dtype}")
    assert tuple(q.shape) == (*lead, (cols + 1) // 2), \
        f"packed weights have shape {tuple(q.shape)}, expected {(*lead, (cols + 1) // 2)}"
    want = (*lead, _groups(cols, G))
    assert isinstance(scale, torch.Tensor) and scale.device == dev, f"scale must be a tensor on {dev}"
    assert tuple(scale.shape) == want, f"scale has shape {tuple(scale.shape)}, expected {want}"
    if zero is not None:
        assert isinstance(zero, torch.Tensor) and zero.device == dev, f"zero must be a tensor on {dev}"
        if zero.dtype is not torch.uint8:
            raise NotImplementedError(f"zero points are uint8, got {zero.dtype}")
        assert tuple(zero.shape) == want, f"zero has shape {tuple(zero.shape)}, expected {want}"
    return _inner(q), _inner(_plain(scale)), _inner(zero)


def _inner(t):
    """t with its last dimension contiguous, no negative or overlapping rows."""
    if t is None:
        return None
    if t.stride(-1) != 1 and t.shape[-1] > 1:
        return t.contiguous()
    if t.dim() >= 2 and t.shape[-2] > 1 and t.stride(-2) < t.shape[-1]:
        return t.contiguous()
    return t


def dequantize_int4(q, scale, group_size=128, *, zero=None, cols=None, out_dtype=torch.bfloat16):
    """The weights ``(u - zero) * scale`` of ``q [..., (cols + 1) // 2]`` as ``[..., cols]`` of
    ``out_dtype`` (fp32, fp16 or bf16): products in fp32, rounded to that type (16-bit scales make
    them exact in fp32).  ``scale`` and the optional uint8 ``zero``
    are ``[..., ceil(cols / group_size)]``; ``cols`` is twice the bytes of a row unless given (an
    odd number of columns has to be).  The result carries no gradient."""
    if isinstance(q, torch.Tensor) and q.dim() == 2:
        out = _try_dequantize(q, scale, zero, 2 * q.shape[1] if cols is None else cols, group_size, out_dtype)
        if out is not None:
            return out
    return _dequantize(q, scale, group_size, zero, cols, out_dtype)


@_on_device
def _dequantize(q, scale, group_size, zero, cols, out_dtype):
    G = _group(group_size)
    if out_dtype not in FLOATS:
        raise NotImplementedError(f"out_dtype must be fp32, fp16 or bf16, got {out_dtype}")
    assert q.dim() >= 1, "dequantize_int4 takes rows"
    cols = 2 * q.shape[-1] if cols is None else int(cols)
    lead, dev = q.shape[:-1], q.device
    q, scale, zero = _check_weight(q, scale, zero, cols, G, lead, dev)
    if scale.dtype not in FLOATS:
        raise NotImplementedError(f"scale must be fp32, fp16 or bf16, got {scale.dtype}")
    rows = lead.numel()
    q2, s2 = _rows(q.reshape(rows, q.shape[-1])), _rows(scale.reshape(rows, scale.shape[-1]))
    z2 = _rows(zero.reshape(rows, zero.shape[-1])) if zero is not None else None
    out = torch.empty((*lead, cols), dtype=out_dtype, device=dev)
    _lib.raise_for(_lib.load().mb_int4_dequantize(
        _lib.DTYPE_CODE[out_dtype], _lib.DTYPE_CODE[scale.dtype], rows, cols, G, q2.data_ptr(), _ld(q2), s2.data_ptr(),
        _ld(s2), z2.data_ptr() if z2 is not None else None, _ld(z2) if z2 is not None else 0, out.data_ptr(), cols,
        _stream_of(dev)), "mb_int4_dequantize")
    return out


def _product(x, q, scale, zero, G, offsets, bias, out, plan):
    d = _lib.Int4Desc()
    M, K = x.shape
    g = q.dim() - 2
    d.dtype, d.scale_dtype, d.group = _lib.DTYPE_CODE[x.dtype], _lib.DTYPE_CODE[scale.dtype], G
    d.bias_dtype = d.dtype
    d.M, d.N, d.K, d.groups = M, q.shape[-2], K, q.shape[0] if g else 0
    d.x, d.x_rs = x.data_ptr(), _ld(x)
    d.w, d.scale, d.out = q.data_ptr(), scale.data_ptr(), out.data_ptr()
    d.w_rs, d.scale_rs = q.stride(-2), scale.stride(-2)
    d.out_rs = _ld(out)
    if g:
        d.w_e, d.scale_e, d.offsets = q.stride(0), scale.stride(0), offsets.data_ptr()
    if zero is not None:
        d.zero, d.zero_rs, d.zero_e = zero.data_ptr(), zero.stride(-2), zero.stride(0) if g else 0
    if bias is not None:
        d.bias, d.bias_dtype = bias.data_ptr(), _lib.DTYPE_CODE[bias.dtype]
    if plan:
        d.plan[:] = plan
    lib = _lib.load()
    need = lib.mb_int4_workspace_size(_byref(d))
    if need > 0:
        # copies of operands that cannot be read in place; the allocator keeps it on this stream
        ws = torch.empty(need, dtype=torch.uint8, device=x.device)
        d.workspace, d.workspace_bytes = ws.data_ptr(), need
    _lib.raise_for(lib.mb_int4_gemm(_byref(d), _stream_of(x.device)), "mb_int4_gemm")


def _check_tokens(x):
    if x.dtype not in TOKENS:
        raise NotImplementedError(f"tokens must be fp16 or bf16, got {x.dtype}")


def _no_derivative(*operands):
    for t in operands:
        if t is None:
            continue
        if t.requires_grad and torch.is_grad_enabled():
            raise NotImplementedError("products with 4-bit weights have no gradient; call under torch.no_grad()")
        if fwd.unpack_dual(t).tangent is not None:
            raise NotImplementedError("products with 4-bit weights have no forward-mode derivative")


def _check_scale_type(scale, x):
    assert isinstance(scale, torch.Tensor), "scale must be a tensor"
    if scale.dtype is not x.dtype and scale.dtype is not torch.float32:
        raise NotImplementedError(f"scale must be {x.dtype} or fp32, got {scale.dtype}")


def _check_out(out, shape, x):
    if out is None:
        return torch.empty(shape, dtype=x.dtype, device=x.device)
    assert isinstance(out, torch.Tensor), "out must be a tensor"
    assert out.device == x.device and tuple(out.shape) == tuple(shape), \
        f"out has shape {tuple(out.shape)} on {out.device}, expected {tuple(shape)} on {x.device}"
    if out.is_neg():
        raise NotImplementedError("out with a lazy negation")
    if out.dtype is not x.dtype:
        raise ValueError(f"out is {out.dtype}, the tokens are {x.dtype}")
    return out


def _out_rows(out, M, N):
    """out as [M, N] rows with contiguous columns."""
    try:
        o = out if out.dim() == 2 else out.view(M, N)
    except RuntimeError:
        raise AssertionError(f"out of shape {tuple(out.shape)} and strides {out.stride()} is no matrix of "
                             "rows") from None
    assert N <= 1 or o.stride(1) == 1, f"out needs contiguous columns, its strides are {out.stride()}"
    if M > 1 and o.stride(0) < N:
        raise ValueError(f"rows of out share memory (strides {out.stride()})")
    return o


def _written(out):
    """Tell autograd: a graph that saved out for its backward pass must not use what stands there now."""
    if not out.is_inference():
        torch.autograd.graph.increment_version(out)


def int4_mm(x, weight, scale, group_size=128, *, zero=None, bias=None, out=None, _plan=None):
    """``x @ w.t() + bias`` for ``x [..., K]`` (fp16 or bf16) and 4-bit weights of N rows of K
    columns: ``weight`` uint8 ``[N, (K + 1) // 2]``, ``scale [N, ceil(K / group_size)]`` of x's
    type or fp32, optional zero points ``zero`` (uint8, like scale), as ``quantize_int4`` makes
    them.  The result ``[..., N]`` has x's type; sums are fp32 and round once.  ``bias [N]`` has
    x's type or fp32.  ``out`` may be any tensor of that shape whose leading dimensions fold
    into rows with contiguous columns that do not overlap; one that shares memory with an operand
    that is read in place is a ValueError.

    Weights are read in place when their rows start on 16-byte boundaries (``quantize_int4``'s
    do); others are copied into scratch in every call.
    """
    if out is None and _plan is None:
        y = _try_int4(x, weight, scale, zero, group_size, None, bias)
        if y is not None:
            return y
    return _int4_mm(x, weight, scale, group_size, zero, bias, out, _plan)


@_on_device
def _int4_mm(x, weight, scale, group_size, zero, bias, out, _plan):
    G = _group(group_size)
    _check_tokens(x)
    assert x.dim() >= 1 and isinstance(weight, torch.Tensor) and weight.dim() == 2, \
        "int4_mm takes x [..., K] and packed weights [N, (K + 1) // 2]"
    K, N, dev = x.shape[-1], weight.shape[0], x.device
    _check_scale_type(scale, x)
    weight, scale, zero = _check_weight(weight, scale, zero, K, G, (N,), dev)
    lead = x.shape[:-1]
    M = lead.numel()
    if bias is not None:
        assert isinstance(bias, torch.Tensor), "bias must be a tensor"
        assert bias.device == dev and tuple(bias.shape) == (N,), f"bias has shape {tuple(bias.shape)}, not ({N},)"
        if bias.dtype is not x.dtype and bias.dtype is not torch.float32:
            raise NotImplementedError(f"bias must be {x.dtype} or fp32, got {bias.dtype}")
        bias = _plain(bias).contiguous()
    out = _check_out(out, (*lead, N), x)
    _no_derivative(x, scale, bias, out)
    _product(_rows(x if x.dim() == 2 else x.reshape(M, K)), weight, scale, zero, G, None, bias, _out_rows(out, M, N),
             _plan)
    _written(out)
    return out


def grouped_int4_mm(x, weight, scale, offsets, group_size=128, *, zero=None, out=None, _plan=None):
    """``int4_mm`` with a weight matrix per group of rows.

    Rows ``offsets[e] .. offsets[e+1]-1`` of ``x [M, K]`` are multiplied with the weights e of
    ``weight [E, N, (K + 1) // 2]``, ``scale`` and ``zero [E, N, ceil(K / group_size)]``; rows at
    or past ``offsets[E]`` come out as zeros.  ``offsets`` is an int32 device tensor of ``E + 1``
    ascending row numbers starting at 0 (``expert_sort``'s): the host never reads it, empty
    groups cost nothing, and E is at most 1024.  Numbers that are not ascending name no groups:
    every row comes out as zeros.
    """
    if out is None and _plan is None and offsets is not None:
        y = _try_int4(x, weight, scale, zero, group_size, offsets, None)
        if y is not None:
            return y
    return _grouped_int4_mm(x, weight, scale, offsets, group_size, zero, out, _plan)


@_on_device
def _grouped_int4_mm(x, weight, scale, offsets, group_size, zero, out, _plan):
    G = _group(group_size)
    _check_tokens(x)
    assert x.dim() == 2 and isinstance(weight, torch.Tensor) and weight.dim() == 3, \
        "grouped_int4_mm takes x [M, K] and packed weights [E, N, (K + 1) // 2]"
    M, K = x.shape
    E, N, dev = weight.shape[0], weight.shape[1], x.device
    if not 1 <= E <= MAX_GROUPS:
        raise ValueError(f"{E} groups: 1 to {MAX_GROUPS} expected")
    assert isinstance(offsets, torch.Tensor), "offsets must be a tensor"
    assert offsets.device == dev and tuple(offsets.shape) == (E + 1,), \
        f"offsets has shape {tuple(offsets.shape)} on {offsets.device}, expected ({E + 1},) on {dev}"
    if offsets.dtype is not torch.int32:
        raise NotImplementedError(f"offsets must be int32, got {offsets.dtype}")
    _check_scale_type(scale, x)
    weight, scale, zero = _check_weight(weight, scale, zero, K, G, (E, N), dev)
    out = _check_out(out, (M, N), x)
    _no_derivative(x, scale, out)
    _product(_rows(x), weight, scale, zero, G, offsets.contiguous(), None, _out_rows(out, M, N), _plan)
    _written(out)
    return out
