"""A mixture-of-experts feed-forward layer on this package's operators.

    python examples/moe_layer.py                       # serving: int8 experts, and a training step
    python examples/moe_layer.py --tokens 1 --top-k 8  # one decoded token

Serving (``Int8Experts``): the router's choices are sorted on the device, the tokens' rows are
quantized on their way into expert order, both projections run as int8 products by expert, and
the weighted rows return to their tokens.  No count is read back to the host, so the whole
layer can be captured in a CUDA graph.

    ids, weights = router(x)                            # [T, k]
    order = expert_sort(ids, E)
    q, s = expert_gather_quantize(x, order)
    h = silu(grouped_scaled_mm(q, up, s, up_scale, order.offsets))
    y = grouped_scaled_mm(*quantize(h)..., down, ..., order.offsets)
    out = expert_combine(y, weights, order)

Training (``train_step``): the same layer in floats; sort, gather and combine take part in
autograd, the experts' products are the framework's ``matmul``.
"""
from __future__ import annotations

import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import metalblas_b200 as mb  # noqa: E402


def route(x, gate, k):
    """Each token's k experts and their weights, by the router's scores."""
    top, ids = torch.topk(x.float() @ gate.float(), k, dim=1)
    return ids, torch.softmax(top, dim=1)


class Int8Experts:
    """Experts' weights ``up [E, hidden, dim]`` and ``down [E, dim, hidden]`` in int8, a scale
    for each output channel."""

    def __init__(self, up, down):
        self.experts = up.shape[0]
        self.up, self.up_scale = mb.quantize(up)
        self.down, self.down_scale = mb.quantize(down)

    def __call__(self, x, ids, weights):
        order = mb.expert_sort(ids, self.experts)
        q, scale = mb.expert_gather_quantize(x, order)
        h = mb.grouped_scaled_mm(q, self.up.transpose(1, 2), scale, self.up_scale, order.offsets, out_dtype=x.dtype)
        q, scale = mb.quantize(torch.nn.functional.silu(h))
        y = mb.grouped_scaled_mm(q, self.down.transpose(1, 2), scale, self.down_scale, order.offsets,
                                 out_dtype=x.dtype)
        return mb.expert_combine(y, weights, order)


class _Product(torch.autograd.Function):
    """``a @ b`` by the framework's matmul, with its gradients."""

    @staticmethod
    def forward(ctx, a, b):
        ctx.save_for_backward(a, b)
        return mb.matmul(a, b)

    @staticmethod
    def backward(ctx, grad):
        a, b = ctx.saved_tensors
        return mb.matmul(grad, b.t()), mb.matmul(a.t(), grad)


def float_layer(x, ids, weights, up, down):
    """The layer in floats, differentiable: rows by expert, a product per expert."""
    order = mb.expert_sort(ids, up.shape[0])
    rows = mb.expert_gather(x, order)
    ends = order.offsets.tolist()
    parts = []
    for e in range(up.shape[0]):
        r = rows[ends[e]:ends[e + 1]]
        if r.shape[0]:
            parts.append(_Product.apply(torch.nn.functional.silu(_Product.apply(r, up[e].t())), down[e].t()))
    parts.append(rows[ends[-1]:, :1].expand(-1, down.shape[1]) * 0)
    return mb.expert_combine(torch.cat(parts).to(x.dtype), weights, order)


def train_step(x, ids, weights, up, down, grad):
    """out and the gradients of x, weights, up and down for the output's gradient."""
    inputs = [t.detach().requires_grad_() for t in (x, weights, up, down)]
    out = float_layer(inputs[0], ids, inputs[1], inputs[2], inputs[3])
    out.backward(grad)
    return out.detach(), [t.grad for t in inputs]


def plain_layer(x, ids, weights, up, down):
    """The layer with torch operations in the inputs' type, every expert on every token."""
    h = torch.nn.functional.silu(torch.einsum("td,ehd->teh", x, up))
    y = torch.einsum("teh,edh->ted", h, down)
    share = torch.zeros(x.shape[0], up.shape[0], dtype=y.dtype, device=x.device).scatter(1, ids, weights.to(y.dtype))
    return (y * share[..., None]).sum(1)


def make(tokens, dim, hidden, experts, k, dtype, device, seed=0):
    g = torch.Generator(device=device).manual_seed(seed)
    rand = lambda *s: torch.randn(s, generator=g, device=device)  # noqa: E731
    x, gate = rand(tokens, dim).to(dtype), rand(dim, experts) / dim ** 0.5
    up = (rand(experts, hidden, dim) / dim ** 0.5).to(dtype)
    down = (rand(experts, dim, hidden) / hidden ** 0.5).to(dtype)
    return x, *route(x, gate, k), up, down, rand(tokens, dim).to(dtype)


def relative_error(a, b):
    a, b = a.detach().double(), b.detach().double()
    return float((a - b).norm() / b.norm())


def main():
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--tokens", type=int, default=256)
    ap.add_argument("--dim", type=int, default=1024)
    ap.add_argument("--hidden", type=int, default=2048)
    ap.add_argument("--experts", type=int, default=16)
    ap.add_argument("--top-k", type=int, default=2)
    a = ap.parse_args()
    x, ids, weights, up, down, grad = make(a.tokens, a.dim, a.hidden, a.experts, a.top_k, torch.bfloat16, "cuda")
    want = plain_layer(x.float(), ids, weights, up.float(), down.float())
    layer = Int8Experts(up, down)
    out = layer(x, ids, weights)
    print(f"int8 experts: relative error {relative_error(out, want):.2e} against fp32")
    start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        layer(x, ids, weights)
    graph.replay()
    start.record()
    for _ in range(20):
        graph.replay()
    end.record()
    end.synchronize()
    print(f"int8 experts: {start.elapsed_time(end) / 20 * 1e3:.1f} us a layer of {a.tokens} tokens (graph replay)")
    out, grads = train_step(x, ids, weights, up, down, grad)
    leaves = [t.detach().float().requires_grad_() for t in (x, weights, up, down)]
    plain = plain_layer(leaves[0], ids, leaves[1], leaves[2], leaves[3])
    plain.backward(grad.float())
    print(f"training step: relative error {relative_error(out, plain):.2e}; gradients " + ", ".join(
        f"{n} {relative_error(g, t.grad):.2e}" for n, g, t in zip(("x", "weights", "up", "down"), grads, leaves)))


if __name__ == "__main__":
    main()
