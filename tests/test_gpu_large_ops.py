"""Operands and results past 2^31 elements: what lies at their far end, on sampled rows."""
from __future__ import annotations

import pytest
import torch

import metalblas_b200 as mb
from metalblas_b200 import kernels
from tests.test_gpu_experts import close
from tests.test_gpu_quantized import check_product

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(autouse=True)
def alone():
    yield
    assert kernels.device_status() == 0
    torch.cuda.empty_cache()


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def ints(shape, g):
    return torch.randint(-127, 128, shape, dtype=torch.int8, generator=g, device=DEV)


def scales(shape, g):
    return torch.rand(shape, generator=g, device=DEV) * 0.02 + 1e-3


@pytest.mark.parametrize("K", [4096, 4095])   # 4095: rows off 16 bytes, copied first
def test_weights_by_group(K):
    g = gen(K)
    E, N = 70, 8192
    W, sb = ints((E, N, K), g), scales((E, N), g)
    assert W.numel() > 1 << 31
    for counts in ({69: 3}, {0: 1, 33: 2, 69: 2}, {0: 20, 69: 21}, {1: 150, 68: 40, 69: 140}):
        M = sum(counts.values())
        a, sa = ints((M, K), g), scales((M,), g)
        off, at = [0], 0
        for e in range(E):
            at += counts.get(e, 0)
            off.append(at)
        y = mb.grouped_scaled_mm(a, W.transpose(1, 2), sa, sb, torch.tensor(off, dtype=torch.int32, device=DEV),
                                 out_dtype=torch.float32)
        for e in counts:
            r = slice(off[e], off[e + 1])
            check_product(y[r], a[r], W[e].t(), sa[r], sb[e])


@pytest.mark.parametrize("N", [32800, 32801])   # 32801: rows of C off 16 bytes
def test_results(N):
    g = gen(N)
    M, K = 66000, 64
    a, sa, w, sb = ints((M, K), g), scales((M,), g), ints((N, K), g).t(), scales((N,), g)
    y = mb.scaled_mm(a, w, sa, sb)
    assert y.numel() > 1 << 31
    for r in (slice(0, 40), slice(65400, 65600), slice(M - 200, M)):
        check_product(y[r], a[r], w, sa[r], sb)


@pytest.mark.parametrize("start", [0, 1])   # 1: rows off 16 bytes, copied first
def test_rows_of_a(start):
    g = gen(start)
    M, K, N = 270000, 8192, 64
    A, sa = ints((M, K), g), scales((M,), g)
    assert A.numel() > 1 << 31
    a = A[:, start:]
    w, sb = ints((N, K), g).t()[:K - start], scales((N,), g)
    y = mb.scaled_mm(a, w, sa, sb, out_dtype=torch.float32)
    for r in (slice(0, 40), slice(262100, 262200), slice(M - 100, M)):
        check_product(y[r], a[r], w, sa[r], sb)


@pytest.mark.parametrize("H", [4096, 4097])   # 4097: rows off 16 bytes
def test_routing(H):
    g = gen(H)
    T, k, E = 262200, 2, 16
    o = mb.expert_sort(torch.randint(-1, E, (T, k), generator=g, device=DEV), E)
    x = torch.randn(T, H, generator=g, device=DEV, dtype=torch.bfloat16)
    kept = int(o.offsets[-1])
    xs = mb.expert_gather(x, o)
    assert xs.numel() > 1 << 31
    n = T * k
    some = torch.cat([torch.arange(0, n, 9973), torch.arange(kept - 300, kept + 300), torch.arange(n - 300, n)]).to(DEV)
    live = (some < kept)[:, None]
    token = (o.order[some] // k).long()
    assert torch.equal(xs[some], torch.where(live, x[token], 0))
    q, s = mb.expert_gather_quantize(x, o)
    wq, ws = mb.quantize(x[token])
    assert torch.equal(q[some], torch.where(live, wq, 0)) and torch.equal(s[some], torch.where(live[:, 0], ws, 0))
    del q, s
    w = torch.rand(T, k, generator=g, device=DEV)
    t = torch.cat([torch.arange(0, T, 9973), torch.arange(T - 300, T)]).to(DEV)
    part = o._replace(position=o.position[t])
    # tokens alone: the sums do not depend on the tokens beside them
    rows = torch.where((part.position < kept)[..., None], xs[part.position.long()], 0).reshape(-1, H)
    alone = mb.ExpertOrder(None, torch.arange(t.numel() * k, dtype=torch.int32, device=DEV).reshape(-1, k),
                           torch.tensor([0, t.numel() * k], dtype=torch.int32, device=DEV))
    out = mb.expert_combine(xs, w, o)
    assert torch.equal(out[t], mb.expert_combine(rows, w[t], alone))
    assert torch.equal(mb.expert_gather_backward(xs, o)[t], mb.expert_gather_backward(rows, alone))
    dy, dw = mb.expert_combine_backward(x, xs, w, o)
    pdy, _ = mb.expert_combine_backward(x[t], rows, w[t], alone)
    p = rows.reshape(-1, k, H).double() * x[t].double()[:, None]
    close(dw[t], p.sum(-1), p.abs().sum(-1), H + 1)   # (rows off 16 bytes: in an order by their place)
    gone = (part.position >= kept).reshape(-1, 1)
    assert torch.equal(dy[part.position.long().reshape(-1)], torch.where(gone, 0, pdy))


@pytest.mark.parametrize("cols", [8200, 8201])
def test_quantize(cols):
    g = gen(cols)
    rows = 262200
    x = torch.randn(rows, cols, generator=g, device=DEV, dtype=torch.bfloat16)
    assert x.numel() > 1 << 31
    q, s = mb.quantize(x)
    r = torch.cat([torch.arange(0, rows, 9973), torch.arange(rows - 300, rows)]).to(DEV)
    wq, ws = mb.quantize(x[r])
    assert torch.equal(q[r], wq) and torch.equal(s[r], ws)
