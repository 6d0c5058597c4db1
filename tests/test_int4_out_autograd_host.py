"""CPU: an ``out`` of the 4-bit products and what autograd knows of it.

The library's entries stand aside (nothing is launched): what counts is which calls reach them, and
what the tensors say of themselves afterwards."""
from __future__ import annotations

import pytest
import torch
import torch.autograd.forward_ad as fwd

from metalblas_b200 import _lib, int4

X, Q, S = torch.zeros(4, 64, dtype=torch.bfloat16), torch.zeros(8, 32, dtype=torch.uint8), torch.ones(8, 2)
OFF = torch.tensor([0, 4], dtype=torch.int32)
CALLS = [lambda out, x=X: int4._int4_mm.__wrapped__(x, Q, S, 32, None, None, out, None),
         lambda out, x=X: int4._grouped_int4_mm.__wrapped__(x, Q[None], S[None], OFF, 32, None, out, None)]


class Library:
    def __init__(self):
        self.launched = 0

    def mb_int4_workspace_size(self, d):
        return 0

    def mb_int4_gemm(self, d, stream):
        self.launched += 1
        return _lib.MB_OK


@pytest.fixture
def library(monkeypatch):
    library = Library()
    monkeypatch.setattr(_lib, "load", lambda: library)
    monkeypatch.setattr(int4, "_stream_of", lambda device: None)
    return library


@pytest.mark.parametrize("call", CALLS)
def test_an_out_that_wants_a_gradient(library, call):
    leaf = torch.empty(4, 8, dtype=torch.bfloat16, requires_grad=True)
    for out in (leaf, leaf * 1):
        with pytest.raises(NotImplementedError, match="no gradient"):
            call(out)
    with fwd.dual_level(), pytest.raises(NotImplementedError, match="forward-mode"):
        call(fwd.make_dual(torch.empty(4, 8, dtype=torch.bfloat16), torch.ones(4, 8, dtype=torch.bfloat16)))
    assert library.launched == 0
    with torch.no_grad():
        assert call(leaf) is leaf
    assert library.launched == 1


@pytest.mark.parametrize("call", CALLS)
def test_a_backward_pass_learns_of_the_write(library, call):
    """What a graph has saved is not the same after the call."""
    buf = torch.ones(4, 8, dtype=torch.bfloat16)
    leaf = torch.ones(4, 8, dtype=torch.bfloat16, requires_grad=True)
    loss = (leaf * buf).sum()
    call(buf)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    with torch.inference_mode():
        call(torch.empty(4, 8, dtype=torch.bfloat16))


@pytest.mark.parametrize("call", CALLS)
def test_a_lazy_negation(library, call):
    """The kernels write values, not their negatives."""
    with pytest.raises(NotImplementedError, match="negation"):
        call(torch.empty(4, 8, dtype=torch.bfloat16)._neg_view())
    assert library.launched == 0
