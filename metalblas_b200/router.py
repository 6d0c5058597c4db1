"""A router's scores to experts and weights, and the loss that keeps the experts in balance.

    weights, experts = expert_route(logits, k)            # logits [T, E]
    order = expert_sort(experts, E)                       # ... the experts' products ...
    out = expert_combine(rows, weights, order)
    balance = expert_balance(logits, experts)
    loss = task_loss + 0.01 * balance.loss

``expert_route``'s weights and ``expert_balance``'s loss take part in reverse-mode autograd, once;
a tangent (forward mode) raises NotImplementedError.  ``expert_route_backward`` and
``expert_balance_backward`` are the gradients by themselves; what they return carries none.
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from . import _lib
from .dispatch import FLOATS, _plain, _stream_of
from .experts import MAX_EXPERTS, _no_tangent
from .quantized import _ld, _on_device, _rows

MAX_K = 64
_WHAT = "expert_route, expert_balance"   # in messages

# The host fast path (csrc/fastops.h): the result of a plain call, or None.
_try_route = _lib.fast_op("try_route")
_try_route_backward = _lib.fast_op("try_route_backward")
_try_balance = _lib.fast_op("try_balance")
_try_balance_backward = _lib.fast_op("try_balance_backward")


class ExpertBalance(NamedTuple):
    """loss    fp32 scalar
    counts  [E] int32, the entries of each expert
    tokens  int32 scalar, the tokens counted"""
    loss: torch.Tensor
    counts: torch.Tensor
    tokens: torch.Tensor


def _check_logits(logits):
    if logits.dtype not in FLOATS:
        raise NotImplementedError(f"logits must be fp32, fp16 or bf16, got {logits.dtype}")
    assert logits.dim() == 2, f"logits must be [tokens, experts], got {tuple(logits.shape)}"
    if not 1 <= logits.shape[1] <= MAX_EXPERTS:
        raise ValueError(f"{logits.shape[1]} experts: 1 to {MAX_EXPERTS} expected")
    return _rows(logits)


def _check_ids(experts, T, dev):
    assert isinstance(experts, torch.Tensor), "experts must be a tensor"
    assert experts.device == dev and experts.dim() == 2 and experts.shape[0] == T, \
        f"experts have shape {tuple(experts.shape)} on {experts.device}, expected [{T}, k] on {dev}"
    if experts.dtype not in (torch.int32, torch.int64):
        raise NotImplementedError(f"expert numbers must be int32 or int64, got {experts.dtype}")
    if experts.dtype is torch.int64:
        # numbers past 32 bits are no expert's
        experts = torch.where((experts >= 0) & (experts < MAX_EXPERTS), experts, -1).to(torch.int32)
    return experts.contiguous()


def _check_mask(mask, T, dev):
    if mask is None:
        return None
    assert isinstance(mask, torch.Tensor), "mask must be a tensor"
    assert mask.device == dev and tuple(mask.shape) == (T,), f"mask has shape {tuple(mask.shape)}, expected ({T},)"
    if mask.dtype is not torch.bool:
        raise NotImplementedError(f"mask must be bool, got {mask.dtype}")
    return mask.contiguous()


def _check_grad(grad, shape, dev):
    assert isinstance(grad, torch.Tensor), "grad must be a tensor"
    assert grad.device == dev and tuple(grad.shape) == tuple(shape), \
        f"grad has shape {tuple(grad.shape)}, expected {tuple(shape)}"
    if grad.dtype is not torch.float32:
        raise NotImplementedError(f"grad must be fp32, got {grad.dtype}")
    return _plain(grad).contiguous()


@_on_device
def _route(logits, k, normalize):
    x = _check_logits(logits)
    T, E = x.shape
    if not 1 <= k <= min(E, MAX_K):
        raise ValueError(f"k = {k} of {E} experts: 1 to {min(E, MAX_K)} expected")
    weights = torch.empty((T, k), dtype=torch.float32, device=x.device)
    experts = torch.empty((T, k), dtype=torch.int32, device=x.device)
    _lib.raise_for(_lib.load().mb_expert_route(_lib.DTYPE_CODE[x.dtype], T, E, k, int(bool(normalize)), x.data_ptr(),
                                               _ld(x), weights.data_ptr(), experts.data_ptr(), _stream_of(x.device)),
                   "mb_expert_route")
    return weights, experts


class _Route(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, k, normalize):
        weights, experts = _route(logits, k, normalize)
        ctx.save_for_backward(logits, experts)
        ctx.normalize = normalize
        ctx.mark_non_differentiable(experts)
        return weights, experts

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad, _):
        _no_tangent(grad, what=_WHAT)
        logits, experts = ctx.saved_tensors
        return expert_route_backward(grad, logits, experts, normalize=ctx.normalize), None, None


def expert_route(logits, k, *, normalize=True):
    """The k experts of each token and their weights: fp32 ``weights [T, k]`` and int32
    ``experts [T, k]`` from ``logits [T, E]`` (fp32, fp16 or bf16; E at most 1024, k at most 64).

    The experts are those of the k largest scores, in descending order, equal ones by their
    numbers; the weights are the softmax over all E scores there, with ``normalize`` divided by
    their sum.  A score of -inf is never chosen: an entry for which no other is left has the
    number -1 (``expert_sort`` drops it) and weight 0.  A NaN counts as the largest score; it
    and +inf make the token's weights NaN.  The weights take part in reverse-mode autograd.
    """
    fast = _try_route(logits, k, normalize)
    if fast is not None:
        return fast
    _no_tangent(logits, what=_WHAT)
    if isinstance(logits, torch.Tensor) and logits.requires_grad and torch.is_grad_enabled():
        return _Route.apply(logits, k, normalize)
    return _route(logits, k, normalize)


def expert_route_backward(grad, logits, experts, *, normalize=True):
    """Gradient of ``expert_route`` by the logits, of their type, from fp32 ``grad [T, k]`` and the
    call's own logits and experts.  Entries outside 0..E-1 contribute nothing.  The result
    carries no gradient."""
    out = _try_route_backward(logits, grad, experts, normalize)
    return out if out is not None else _route_backward(logits, grad, experts, normalize)


@_on_device
def _route_backward(logits, grad, experts, normalize):
    x = _check_logits(logits)
    T, E = x.shape
    ids = _check_ids(experts, T, x.device)
    grad = _check_grad(grad, ids.shape, x.device)
    out = torch.empty((T, E), dtype=x.dtype, device=x.device)
    _lib.raise_for(_lib.load().mb_expert_route_backward(
        _lib.DTYPE_CODE[x.dtype], T, E, ids.shape[1], int(bool(normalize)), grad.data_ptr(), x.data_ptr(), _ld(x),
        ids.data_ptr(), out.data_ptr(), _stream_of(x.device)), "mb_expert_route_backward")
    return out


@_on_device
def _balance(logits, experts, mask):
    x = _check_logits(logits)
    T, E = x.shape
    dev = x.device
    ids, mask = _check_ids(experts, T, dev), _check_mask(mask, T, dev)
    loss = torch.empty((), dtype=torch.float32, device=dev)
    counts = torch.empty(E, dtype=torch.int32, device=dev)
    tokens = torch.empty((), dtype=torch.int32, device=dev)
    lib = _lib.load()
    ws = torch.empty(lib.mb_expert_balance_workspace_size(T, E), dtype=torch.uint8, device=dev)
    _lib.raise_for(lib.mb_expert_balance(
        _lib.DTYPE_CODE[x.dtype], T, E, ids.shape[1], x.data_ptr(), _ld(x), ids.data_ptr(),
        mask.data_ptr() if mask is not None else None, loss.data_ptr(), counts.data_ptr(), tokens.data_ptr(),
        ws.data_ptr(), ws.numel(), _stream_of(dev)), "mb_expert_balance")
    return loss, counts, tokens


class _Balance(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, experts, mask):
        loss, counts, tokens = _balance(logits, experts, mask)
        ctx.save_for_backward(logits, counts, tokens, mask)
        ctx.mark_non_differentiable(counts, tokens)
        return loss, counts, tokens

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad, _, __):
        _no_tangent(grad, what=_WHAT)
        logits, counts, tokens, mask = ctx.saved_tensors
        return expert_balance_backward(grad, logits, ExpertBalance(None, counts, tokens), mask=mask), None, None


def expert_balance(logits, experts, mask=None):
    """``ExpertBalance(loss, counts, tokens)`` of a router's ``logits [T, E]`` and the ``experts
    [T, k]`` (int32 or int64) chosen from them.

    ``counts[e]`` is the number of entries of expert e, numbers outside 0..E-1 left out;
    ``loss = E * sum_e (counts[e] / sum(counts)) * mean_t softmax(logits[t])[e]``: 1 when the
    load is even, up to E when one expert has it all.  ``mask [T]`` (bool) names the tokens that
    count, for instance those that are no padding; without one the loss is 0.  A row of -inf
    alone has no probabilities and adds nothing.  The loss takes part in reverse-mode autograd
    (the counts are constants).
    """
    fast = _try_balance(logits, experts, mask)
    if fast is not None:
        return ExpertBalance(*fast)
    _no_tangent(logits, what=_WHAT)
    if isinstance(logits, torch.Tensor) and logits.requires_grad and torch.is_grad_enabled():
        return ExpertBalance(*_Balance.apply(logits, experts, mask))
    return ExpertBalance(*_balance(logits, experts, mask))


def expert_balance_backward(grad, logits, balance, mask=None):
    """Gradient of ``expert_balance``'s loss by the logits, of their type, from the fp32 scalar
    ``grad`` and the call's own logits, mask and result.  The result carries no gradient."""
    out = _try_balance_backward(logits, grad, balance.counts, balance.tokens, mask)
    return out if out is not None else _balance_backward(logits, grad, balance, mask)


@_on_device
def _balance_backward(logits, grad, balance, mask):
    x = _check_logits(logits)
    T, E = x.shape
    dev = x.device
    mask, grad = _check_mask(mask, T, dev), _check_grad(grad, (), dev)
    counts, tokens = balance.counts, balance.tokens
    assert isinstance(counts, torch.Tensor) and isinstance(tokens, torch.Tensor), "balance holds tensors"
    assert counts.device == dev and tuple(counts.shape) == (E,) and tokens.device == dev and tokens.dim() == 0, \
        f"counts have shape {tuple(counts.shape)}, expected ({E},)"
    if counts.dtype is not torch.int32 or tokens.dtype is not torch.int32:
        raise NotImplementedError("ExpertBalance holds int32 counts")
    counts = counts.contiguous()   # (named: a copy has to live until the launch)
    out = torch.empty((T, E), dtype=x.dtype, device=dev)
    _lib.raise_for(_lib.load().mb_expert_balance_backward(
        _lib.DTYPE_CODE[x.dtype], T, E, grad.data_ptr(), x.data_ptr(), _ld(x), counts.data_ptr(),
        tokens.data_ptr(), mask.data_ptr() if mask is not None else None, out.data_ptr(), _stream_of(dev)),
        "mb_expert_balance_backward")
    return out
