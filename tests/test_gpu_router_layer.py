"""The router, the 4-bit experts and their plumbing as a layer uses them: served (eager, and
replayed from a graph over new tokens) and trained.

Bounds: a bf16 value is off by 2^-8 of it at most when it is stored.  The served layer stores
the rows' first product, its activation, the second product and the result, each off by that at
most (errors pass through the second product with the norm of what they belong to): 4 roundings,
2 % of the norm is more than four times 2^-8.  The training step stores as many in each direction
(12 between the output's gradient and the tokens'): 5 %.  The gate is fp32; its gradient's terms come
through the output rows' products with the gradient, off by 2^-8 of what is multiplied.
"""
from __future__ import annotations

import os
import sys

import pytest
import torch

import metalblas_b200 as mb

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))
import moe_layer  # noqa: E402

pytestmark = pytest.mark.gpu
SIZES = [(1, 128, 256, 4, 2), (64, 256, 512, 8, 2), (300, 272, 400, 6, 3)]


@pytest.mark.parametrize("tokens,dim,hidden,experts,k", SIZES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_served(tokens, dim, hidden, experts, k, dtype):
    x, _, _, up, down, _ = moe_layer.make(tokens, dim, hidden, experts, k, dtype, "cuda")
    gate = moe_layer.make_gate(dim, experts, "cuda").to(dtype)
    layer = moe_layer.Int4Experts(up, down, 64)

    def step():
        scores = mb.matmul(x, gate)
        weights, ids = mb.expert_route(scores, k)
        return layer(x, ids, weights), ids, weights

    def check(out, ids, weights):
        want = moe_layer.plain_layer(x.double(), ids.long(), weights.double(), *(w.double() for w in layer.floats(torch.float32)))
        assert moe_layer.relative_error(out, want) < 0.02

    first = step()
    check(*first)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        again = step()
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(first, again))
    x.copy_(torch.randn(tokens, dim, generator=torch.Generator().manual_seed(5)).to(dtype))
    graph.replay()
    check(*again)
    assert all(torch.equal(a, b) for a, b in zip(step(), again))


@pytest.mark.parametrize("tokens,dim,hidden,experts,k", SIZES)
def test_trained(tokens, dim, hidden, experts, k):
    x, _, _, up, down, grad = moe_layer.make(tokens, dim, hidden, experts, k, torch.bfloat16, "cuda")
    gate = moe_layer.make_gate(dim, experts, "cuda")
    out, balance, ids, grads = moe_layer.train_router_step(x, gate, up, down, k, grad, balance=0.5)
    leaves = [t.detach().double().requires_grad_() for t in (x, gate, up, down)]
    want, loss = moe_layer.plain_router_layer(*leaves, ids.long())
    torch.autograd.backward([want, loss], [grad.double(), torch.full_like(loss, 0.5)])
    assert moe_layer.relative_error(out, want) < 0.02
    assert abs(float(balance) - float(loss)) < 1e-4 * float(loss)
    for g, t in zip(grads, leaves):
        assert moe_layer.relative_error(g, t.grad) < 0.05


def test_example_runs(monkeypatch, capsys):
    monkeypatch.setattr(sys, "argv", ["moe_layer.py", "--tokens", "40", "--dim", "128", "--hidden", "192", "--experts", "4"])
    moe_layer.main()
    text = capsys.readouterr().out
    assert "4-bit experts" in text and "with its router" in text


def test_training_step_in_a_graph():
    """Forward and backward of a step captured together; the gradient goes on with new scores."""
    T, E, k = 96, 16, 2
    g = torch.Generator().manual_seed(7)
    scores = torch.randn(T, E, generator=g).cuda().requires_grad_()
    up = torch.randn(T, k, generator=g).cuda()

    def step():
        w, ids = mb.expert_route(scores, k, normalize=False)
        loss = (w * up).sum() + mb.expert_balance(scores, ids).loss
        return torch.autograd.grad(loss, scores)[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for seed in (1, 2):
        with torch.no_grad():
            scores.copy_(torch.randn(T, E, generator=torch.Generator().manual_seed(seed)))
        graph.replay()
        assert torch.equal(got, step())
