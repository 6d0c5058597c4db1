"""The example layer: int8 serving and a training step against the layer in torch operations.

Bounds: an int8 operand is off by at most half a step, 1/254 of its row's largest value; with
rows and weights of normal values (largest about four deviations) that is about 1 % of the
operand, twice per product, in two products: 4 % of the output's norm is more than their sum in
quadrature.  bf16 training rounds every stored value to 2^-8 of it at most, a handful of times: 2 %.
"""
from __future__ import annotations

import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))
import moe_layer  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("tokens,dim,hidden,experts,k", [(1, 128, 256, 4, 2), (64, 256, 512, 8, 2), (300, 272, 400, 6, 3)])
def test_layer(tokens, dim, hidden, experts, k):
    x, ids, weights, up, down, grad = moe_layer.make(tokens, dim, hidden, experts, k, torch.bfloat16, "cuda")
    want = moe_layer.plain_layer(x.double(), ids, weights.double(), up.double(), down.double())
    layer = moe_layer.Int8Experts(up, down)
    out = layer(x, ids, weights)
    assert moe_layer.relative_error(out, want) < 0.04
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        again = layer(x, ids, weights)
    graph.replay()
    assert torch.equal(again, out)

    got, grads = moe_layer.train_step(x, ids, weights, up, down, grad)
    leaves = [t.detach().double().requires_grad_() for t in (x, weights, up, down)]
    plain = moe_layer.plain_layer(leaves[0], ids, leaves[1], leaves[2], leaves[3])
    plain.backward(grad.double())
    assert moe_layer.relative_error(got, plain) < 0.02
    for g, t in zip(grads, leaves):
        assert moe_layer.relative_error(g, t.grad) < 0.02
