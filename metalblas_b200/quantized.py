"""int8 products with a scale for each token and each output channel.

``quantize`` turns rows of floats into int8 rows with one fp32 scale each;
``scaled_mm`` multiplies int8 matrices on the int8 tensor cores and applies both
scales (and a bias) in the epilogue; ``grouped_scaled_mm`` does so with one weight
matrix per group of rows, the groups given by device-side offsets, as a
mixture-of-experts layer has them after ``expert_sort``.

The products are exact in 32-bit integers and round once, so their result does not
depend on the tile, the split or the number of rows in the call.  They have no
gradient: rounding to int8 has none, and the weights are constants.
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib
from .dispatch import FLOATS, _plain, _stream_of

MAX_K = 131071       # 127 or 128 squared times more would leave 32 bits
MAX_GROUPS = 1024

_byref = ctypes.byref
# The host fast path (csrc/fastops.h): the result of a plain call, or None.
_try_quantize = _lib.fast_op("try_quantize")
_try_scaled = _lib.fast_op("try_scaled")


def _on_device(fn):
    """Run fn with the device of its first argument current."""
    def call(t, *args, **kw):
        assert isinstance(t, torch.Tensor) and t.is_cuda, "CUDA tensors expected"
        if torch.cuda.current_device() != t.device.index:
            with torch.cuda.device(t.device):
                return fn(t, *args, **kw)
        return fn(t, *args, **kw)
    call.__name__, call.__doc__, call.__wrapped__ = fn.__name__, fn.__doc__, fn
    return call


def _rows(x):
    """x with its last dimension contiguous and rows that do not overlap."""
    x = _plain(x)
    if x.stride(-1) == 1 or x.shape[-1] <= 1:
        if x.dim() < 2 or x.shape[0] <= 1 or x.stride(0) >= x.shape[1]:
            return x
    return x.contiguous()


def _ld(x):
    return max(x.stride(0), x.shape[1]) if x.shape[0] > 1 else x.shape[1]


def _int8_rows(rows, cols, device):
    """An int8 matrix whose rows start on 16-byte boundaries, so that a product can
    read it in place (contiguous when cols is a multiple of 16)."""
    pitch = (cols + 15) // 16 * 16
    q = torch.empty((rows, pitch), dtype=torch.int8, device=device)
    return q if pitch == cols else q[:, :cols]


def quantize(x):
    """Rows of ``x [..., cols]`` (fp32, fp16 or bf16) as ``(q, scale)``: int8 ``q`` of x's
    shape and fp32 ``scale`` of its leading dimensions, with ``x ~ q * scale[..., None]``.

    ``scale = max|x| / 127`` of the row and ``q = round(127 x / max|x|)``, halves to even.  A
    row of zeros has scale 0.  A row with an infinity or a NaN has scale NaN and q 0.  The
    rows of a 2-D ``q`` start on 16-byte boundaries: with a number of columns that is no
    multiple of 16, ``q`` is a view of a wider matrix.  Neither carries a gradient.
    """
    return _try_quantize(x) or _quantize(x)


@_on_device
def _quantize(x):
    if x.dtype not in FLOATS:
        raise NotImplementedError(f"quantize takes fp32, fp16 or bf16, got {x.dtype}")
    assert x.dim() >= 1, "quantize takes rows"
    lead, cols = x.shape[:-1], x.shape[-1]
    x2 = _rows(x if x.dim() == 2 else x.reshape(-1, cols) if cols else x.reshape(lead.numel(), 0))
    rows = x2.shape[0]
    q = _int8_rows(rows, cols, x.device)
    scale = torch.empty(rows, dtype=torch.float32, device=x.device)
    _lib.raise_for(_lib.load().mb_quantize(_lib.DTYPE_CODE[x.dtype], rows, cols, x2.data_ptr(), _ld(x2), q.data_ptr(),
                                           max(q.stride(0), cols), scale.data_ptr(), _stream_of(x.device)),
                   "mb_quantize")
    if x.dim() != 2:
        q, scale = q.reshape(x.shape), scale.reshape(lead)
    return q, scale


def _scale(s, shape, name, device):
    """A scale tensor of `shape`, or one that broadcasts to it; fp32 on the device."""
    assert isinstance(s, torch.Tensor) and s.device == device, f"{name} must be a tensor on {device}"
    if s.dtype is not torch.float32:
        raise NotImplementedError(f"{name} must be fp32, got {s.dtype}")
    assert s.dim() <= len(shape), f"{name} has shape {tuple(s.shape)}, not {tuple(shape)}"
    if tuple(s.shape) != tuple(shape):
        assert all(a in (1, b) for a, b in zip(s.shape[::-1], shape[::-1])), \
            f"{name} has shape {tuple(s.shape)}, not {tuple(shape)}"
        s = s.expand(shape)
    return _plain(s)


def _product(a2, b, sa, sb, M, N, K, groups, offsets, bias, out_dtype, c, overrides):
    d = _lib.ScaledDesc()
    code = _lib.DTYPE_CODE[out_dtype]
    d.out_dtype = d.bias_dtype = code
    d.M, d.N, d.K, d.groups = M, N, K, groups
    d.A, d.B, d.C = a2.data_ptr(), b.data_ptr(), c.data_ptr()
    d.a_rs, d.a_cs = a2.stride()
    d.b_rs, d.b_cs = b.stride()[-2:]
    d.c_rs, d.c_cs = c.stride()
    d.scale_a, d.scale_a_s = sa.data_ptr(), sa.stride(0)
    d.scale_b, d.scale_b_s = sb.data_ptr(), sb.stride(-1)
    if groups:
        d.sB, d.scale_b_g = b.stride(0), sb.stride(0)
        d.offsets = offsets.data_ptr()
    if bias is not None:
        d.bias, d.bias_s, d.bias_dtype = bias.data_ptr(), bias.stride(0), _lib.DTYPE_CODE[bias.dtype]
    if overrides:
        d.tile_n, d.split_k, d.swap_ab, d.cta_pair = overrides
    lib = _lib.load()
    stream = _stream_of(c.device)
    need = lib.mb_scaled_workspace_size(_byref(d))
    if need > 0:
        # copies of operands that cannot be read in place; the allocator keeps it on this stream
        ws = torch.empty(need, dtype=torch.uint8, device=c.device)
        d.workspace, d.workspace_bytes = ws.data_ptr(), need
    _lib.raise_for(lib.mb_scaled_gemm(_byref(d), stream), "mb_scaled_gemm")


def _check_int8(a, b):
    if a.dtype is not torch.int8 or b.dtype is not torch.int8:
        raise NotImplementedError(f"int8 operands expected, got {a.dtype} and {b.dtype}")
    assert a.device == b.device, "operands on different devices"
    if a.is_neg() or b.is_neg():
        raise NotImplementedError("int8 operands with a lazy negation")
    if a.shape[-1] > MAX_K:
        raise ValueError(f"K = {a.shape[-1]}: sums of more than {MAX_K} int8 products can leave 32 bits")


def _check_out(out_dtype, out, shape, device):
    if out is not None:
        assert isinstance(out, torch.Tensor), "out must be a tensor"
        assert out.device == device and tuple(out.shape) == tuple(shape), \
            f"out has shape {tuple(out.shape)} on {out.device}, expected {tuple(shape)} on {device}"
        if out_dtype is not None and out.dtype is not out_dtype:
            raise ValueError(f"out is {out.dtype}, out_dtype is {out_dtype}")
        out_dtype = out.dtype
    out_dtype = out_dtype or torch.bfloat16
    if out_dtype not in FLOATS:
        raise NotImplementedError(f"out_dtype must be fp32, fp16 or bf16, got {out_dtype}")
    return out_dtype


def _check_bias(bias, N, out_dtype, device):
    if bias is None:
        return None
    assert isinstance(bias, torch.Tensor), "bias must be a tensor"
    assert bias.device == device and tuple(bias.shape) == (N,), f"bias has shape {tuple(bias.shape)}, not ({N},)"
    if bias.dtype is not out_dtype and bias.dtype is not torch.float32:
        raise NotImplementedError(f"bias must be {out_dtype} or fp32, got {bias.dtype}")
    return _plain(bias)


def scaled_mm(a, b, scale_a, scale_b, *, bias=None, out_dtype=None, out=None, _plan=None):
    """``(a @ b) * scale_a[..., None] * scale_b + bias`` for int8 ``a [..., K]`` and ``b [K, N]``.

    ``scale_a`` has a's leading shape (one scale per token) and ``scale_b [N]`` one scale per
    output channel; either may also be any shape that broadcasts to that, such as a single
    scale.  ``out_dtype`` is bf16 (default), fp16 or fp32; ``bias [N]`` has that type or fp32.
    The sum over K is exact, so K is at most 131071.  ``out`` may have any strides that give
    every element a place of its own and fold its leading dimensions into one.

    ``b`` is read in place when it is row- or column-major (a transposed ``[N, K]`` weight) on
    a 16-byte aligned base and pitch, as is ``a`` with contiguous aligned rows; other layouts
    are copied into scratch in every call.
    """
    if out is None and _plan is None:
        c = _try_scaled(a, b, scale_a, scale_b, None, bias, out_dtype or torch.bfloat16)
        if c is not None:
            return c
    return _scaled_mm(a, b, scale_a, scale_b, bias, out_dtype, out, _plan)


@_on_device
def _scaled_mm(a, b, scale_a, scale_b, bias, out_dtype, out, _plan):
    assert isinstance(b, torch.Tensor) and b.dim() == 2 and a.dim() >= 1, "scaled_mm takes a [..., K] and b [K, N]"
    _check_int8(a, b)
    K, N = b.shape
    assert a.shape[-1] == K, f"inner dimensions differ: {tuple(a.shape)} @ {tuple(b.shape)}"
    lead = a.shape[:-1]
    dev = a.device
    out_dtype = _check_out(out_dtype, out, (*lead, N), dev)
    bias = _check_bias(bias, N, out_dtype, dev)
    sa = _scale(scale_a, lead, "scale_a", dev)
    sb = _scale(scale_b, (N,), "scale_b", dev)
    M = lead.numel()
    a2 = a if a.dim() == 2 else a.reshape(M, K)
    sa = sa.reshape(M) if sa.dim() != 1 else sa
    if out is None:
        out = torch.empty((*lead, N), dtype=out_dtype, device=dev)
    try:
        c = out if out.dim() == 2 else out.view(M, N)
    except RuntimeError:
        raise AssertionError(f"out of shape {tuple(out.shape)} and strides {out.stride()} is no matrix of "
                             "rows") from None
    _product(a2, b, sa, sb, M, N, K, 0, None, bias, out_dtype, c, _plan)
    return out


def grouped_scaled_mm(a, b, scale_a, scale_b, offsets, *, out_dtype=None, out=None, _plan=None):
    """``scaled_mm`` with a weight matrix per group of rows.

    Rows ``offsets[e] .. offsets[e+1]-1`` of int8 ``a [M, K]`` are multiplied with ``b[e]`` of
    ``b [E, K, N]`` and scaled by ``scale_a [M]`` and ``scale_b [E, N]``; rows at or past
    ``offsets[E]`` come out as zeros.  ``offsets`` is an int32 device tensor of ``E + 1``
    ascending row numbers starting at 0 (``expert_sort``'s): the host never reads it, empty
    groups cost nothing, and E is at most 1024.  Numbers that are not ascending name no groups:
    every row comes out as zeros.
    """
    if out is None and _plan is None:
        c = _try_scaled(a, b, scale_a, scale_b, offsets, None, out_dtype or torch.bfloat16)
        if c is not None:
            return c
    return _grouped_scaled_mm(a, b, scale_a, scale_b, offsets, out_dtype, out, _plan)


@_on_device
def _grouped_scaled_mm(a, b, scale_a, scale_b, offsets, out_dtype, out, _plan):
    assert isinstance(b, torch.Tensor) and a.dim() == 2 and b.dim() == 3, \
        "grouped_scaled_mm takes a [M, K] and b [E, K, N]"
    _check_int8(a, b)
    M, K = a.shape
    E, Kb, N = b.shape
    assert K == Kb, f"inner dimensions differ: {tuple(a.shape)} @ {tuple(b.shape)}"
    if not 1 <= E <= MAX_GROUPS:
        raise ValueError(f"{E} groups: 1 to {MAX_GROUPS} expected")
    dev = a.device
    assert isinstance(offsets, torch.Tensor), "offsets must be a tensor"
    assert offsets.device == dev and tuple(offsets.shape) == (E + 1,), \
        f"offsets has shape {tuple(offsets.shape)} on {offsets.device}, expected ({E + 1},) on {dev}"
    if offsets.dtype is not torch.int32:
        raise NotImplementedError(f"offsets must be int32, got {offsets.dtype}")
    out_dtype = _check_out(out_dtype, out, (M, N), dev)
    sa = _scale(scale_a, (M,), "scale_a", dev)
    sb = _scale(scale_b, (E, N), "scale_b", dev)
    if out is None:
        out = torch.empty((M, N), dtype=out_dtype, device=dev)
    _product(a, b, sa, sb, M, N, K, E, offsets.contiguous(), None, out_dtype, out, _plan)
    return out
