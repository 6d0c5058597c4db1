"""What the routing operators do with derivatives they cannot carry: a tangent is refused, not
dropped; second derivatives are refused; the operators without a gradient say so by their result."""
from __future__ import annotations

import pytest
import torch
import torch.autograd.forward_ad as fwd

import metalblas_b200 as mb

pytestmark = pytest.mark.gpu
DEV = "cuda"
T, K, E, H = 12, 2, 5, 40


def make(seed=0):
    g = torch.Generator().manual_seed(seed)
    o = mb.expert_sort(torch.randint(-1, E, (T, K), generator=g).to(DEV), E)
    rand = lambda *s: torch.randn(*s, generator=g).to(DEV)  # noqa: E731
    return o, rand(T, H), rand(T * K, H), rand(T, K)


def test_tangents_are_refused():
    o, x, rows, w = make()
    with fwd.dual_level():
        with pytest.raises(NotImplementedError):
            mb.expert_gather(fwd.make_dual(x, torch.ones_like(x)), o)
        with pytest.raises(NotImplementedError):
            mb.expert_combine(fwd.make_dual(rows, torch.ones_like(rows)), w, o)
        with pytest.raises(NotImplementedError):
            mb.expert_combine(rows, fwd.make_dual(w, torch.ones_like(w)), o)
        with pytest.raises(NotImplementedError):
            mb.expert_combine(fwd.make_dual(rows, torch.ones_like(rows)), None, o)
        # a layout the host fast path does not take
        wide = torch.zeros(T, 2 * H, device=DEV)
        with pytest.raises(NotImplementedError):
            mb.expert_gather(fwd.make_dual(wide, torch.ones_like(wide))[:, ::2], o)
        # and with a gradient recorded beside it
        leaf = x.clone().requires_grad_()
        with pytest.raises((NotImplementedError, RuntimeError)):
            mb.expert_gather(fwd.make_dual(leaf, torch.ones_like(x)), o)
        # no tangent among the operands: as ever
        assert torch.equal(mb.expert_gather(x, o), mb.expert_gather(fwd.unpack_dual(x).primal, o))
    assert torch.equal(mb.expert_combine(rows, w, o), mb.expert_combine(rows.clone(), w, o))


def test_tangents_of_a_gradient_are_refused():
    """Forward over reverse: the tangent comes with the output's gradient."""
    o, x, rows, w = make(3)
    x.requires_grad_()
    rows.requires_grad_()
    for out in (mb.expert_gather(x, o), mb.expert_combine(rows, w, o)):
        with fwd.dual_level():
            d = fwd.make_dual(torch.ones_like(out), torch.ones_like(out))
            with pytest.raises(NotImplementedError):
                torch.autograd.grad(out, [x, rows], d, allow_unused=True)


def test_second_derivatives_are_refused():
    o, x, rows, w = make(1)
    x.requires_grad_()
    (first,) = torch.autograd.grad(mb.expert_gather(x, o).pow(2).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        first.sum().backward()
    rows.requires_grad_()
    (first,) = torch.autograd.grad(mb.expert_combine(rows, w, o).pow(2).sum(), rows, create_graph=True)
    with pytest.raises(RuntimeError):
        first.sum().backward()


def test_results_without_a_gradient():
    """The gradients by themselves and the quantizing operators record nothing."""
    o, x, rows, w = make(2)
    for t in (x, rows, w):
        t.requires_grad_()
    out = [mb.expert_gather_backward(rows, o), *mb.expert_combine_backward(x, rows, w, o), *mb.quantize(x),
           *mb.expert_gather_quantize(x, o)]
    assert not any(t.requires_grad for t in out)
