"""The host fast path of the int8 and expert operators serves the plain call, gives the Python
path's results, and leaves the rest to it."""
from __future__ import annotations

import pytest
import torch

import metalblas_b200 as mb
from metalblas_b200 import _lib, experts, quantized

pytestmark = pytest.mark.gpu
DEV = "cuda"


def equal(a, b):
    return len(a) == len(b) and all(torch.equal(x, y) for x, y in zip(a, b))


def test_plain_calls_are_served():
    fast = _lib.fast()
    assert fast is not None
    g = torch.Generator().manual_seed(3)
    T, k, E, K, N = 20, 2, 4, 64, 48
    ids = torch.randint(-1, E, (T, k), generator=g).to(DEV)
    x, w = torch.randn(T, K, generator=g).to(DEV), torch.randn(E, N, K, generator=g).to(DEV)
    order = fast.try_sort(ids, E)
    assert order is not None and equal(order, experts._sort(ids, E))
    o = mb.ExpertOrder(*order)
    q = fast.try_quantize(x)
    assert q is not None and equal(q, quantized._quantize(x))
    wq, sw = mb.quantize(w)
    y = fast.try_scaled(q[0], wq[0].t(), q[1], sw[0], None, None, torch.float32)
    assert y is not None and torch.equal(y, quantized._scaled_mm(q[0], wq[0].t(), q[1], sw[0], None, torch.float32,
                                                                 None, None))
    rows = fast.try_gather(x, o.position, o.offsets)
    assert rows is not None and torch.equal(rows, experts._gather(x, o))
    gq = fast.try_gather_quantize(x, o.position, o.offsets)
    assert gq is not None and equal(gq, experts._gather_quantize(x, o))
    z = fast.try_scaled(gq[0], wq.transpose(1, 2), gq[1], sw, o.offsets, None, torch.float32)
    assert z is not None and torch.equal(z, quantized._grouped_scaled_mm(gq[0], wq.transpose(1, 2), gq[1], sw,
                                                                         o.offsets, torch.float32, None, None))
    weights = torch.rand(T, k, generator=g).to(DEV)
    for wt in (weights, None):
        out = fast.try_combine(z, wt, o.position, o.offsets)
        assert out is not None and torch.equal(out, experts._combine(z, wt, o))
    both = fast.try_combine_backward(out, z, weights, o.position, o.offsets)
    assert both is not None and equal(both, experts._combine_backward(out, z, weights, o))
    # what it does not take
    assert fast.try_quantize(x.double()) is None and fast.try_quantize(x.tolist()) is None
    assert fast.try_scaled(q[0], wq[0].t(), 1.0, sw[0], None, None, torch.float32) is None
    with pytest.raises(AssertionError, match="scale_a"):
        mb.scaled_mm(q[0], wq[0].t(), 1.0, sw[0])
