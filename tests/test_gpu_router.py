"""The router and its balance loss, with gradients, against their formulas in 64 bits.

Bounds: an exponential of y <= 0 is within |y| / 2 + 2 units of 2^-23 of its value and a division
within 2, a sum of n terms within n units of 2^-24 of their sizes; a probability p is an exponential
times the inverse of a sum of E of them.  Errors by |y| count with the size of what they belong to:
p |y| / 2 with y no less than -20 is under 10 units of p, and in the sum, where p is the weight of
each, under ln(E) / 2.  (E + 12) units of 2^-23 of p is more than all of it.
Gradients are sums and products of such values, each of which adds its own unit; results of the
scores' type round once.  The chosen experts and the counts are whole numbers and equal.
"""
from __future__ import annotations

import math

import pytest
import torch

import metalblas_b200 as mb

pytestmark = pytest.mark.gpu
DEV = "cuda"
UNIT = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float32: 2.0 ** -126, torch.float16: 2.0 ** -24, torch.bfloat16: 2.0 ** -126}
FLOATS = (torch.float32, torch.float16, torch.bfloat16)
INF, NAN = math.inf, math.nan


def gen(seed):
    return torch.Generator().manual_seed(seed)


def close(got, want, size, terms):
    u = UNIT[got.dtype]
    tol = terms * 2.0 ** -23 * size + u * want.abs() + TINY[got.dtype]
    err = (got.double() - want).abs()
    assert bool((err <= tol).all()), f"off by {float((err / tol).max())} of the bound"


def softmax(x):
    p = torch.softmax(x.double(), 1)
    return torch.where((x == -INF).all(1, keepdim=True), 0.0, p)


def plain_route(x, k, normalize):
    p = softmax(x)
    ids = torch.argsort(x.double().cpu(), dim=1, descending=True, stable=True)[:, :k].to(x.device)
    usable = torch.gather(x, 1, ids) > -INF
    w = torch.where(usable, torch.gather(p, 1, ids), 0.0)
    if normalize:
        w = w / torch.where(w.sum(1, keepdim=True) == 0, 1.0, w.sum(1, keepdim=True))
    return w, torch.where(usable, ids, -1).to(torch.int32)


CASES = [(1, 1, 1), (1, 8, 2), (3, 4, 4), (16, 64, 8), (33, 60, 6), (50, 32, 32), (100, 128, 8), (77, 100, 3),
         (257, 256, 8), (40, 250, 64), (19, 512, 40), (21, 513, 5), (5000, 16, 2), (12, 1024, 8), (9, 1000, 33)]


@pytest.mark.parametrize("T,E,k", CASES)
@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("normalize", [True, False])
def test_route_and_gradient(T, E, k, dtype, normalize):
    g = gen(T + E + k)
    x = (torch.randn(T, E, generator=g) * 2).to(dtype)
    x = torch.where(torch.rand(T, E, generator=g) < 0.2, torch.tensor(-INF, dtype=dtype), x).to(DEV)
    x[T // 2] = -INF
    grad = torch.randn(T, k, generator=g).to(DEV)
    w, ids = mb.expert_route(x, k, normalize=normalize)
    want, want_ids = plain_route(x, k, normalize)
    assert torch.equal(ids, want_ids) and w.dtype is torch.float32
    close(w, want, want, E + k + 12)
    d = mb.expert_route_backward(grad, x, ids, normalize=normalize)
    hot = torch.zeros(T, k, E, dtype=torch.float64, device=DEV)
    hot.scatter_(2, ids.clamp_min(0).long()[..., None], 1.0)
    hot *= (ids >= 0)[..., None]
    G = grad.double()
    mean, size = (want * G).sum(1, keepdim=True), (want * G).abs().sum(1, keepdim=True)
    p = softmax(x)
    if normalize:
        dl = torch.einsum("tke,tk->te", hot, want * (G - mean))
        sz = torch.einsum("tke,tk->te", hot, want * (G.abs() + size))
    else:
        dl = torch.einsum("tke,tk->te", hot, want * G) - p * mean
        sz = torch.einsum("tke,tk->te", hot, want * G.abs()) + p * size
    assert d.dtype is dtype
    close(d, dl, sz, 2 * (E + k) + 32)


@pytest.mark.parametrize("normalize", [True, False])
def test_route_gradient_by_differences(normalize):
    """Central differences of the 64-bit formula with the chosen experts held."""
    x = torch.randn(6, 10, generator=gen(1)).to(DEV)
    w, ids = mb.expert_route(x, 3, normalize=normalize)
    g = torch.randn(6, 3, generator=gen(2)).to(DEV)
    d = mb.expert_route_backward(g, x, ids, normalize=normalize).double()

    def f(y):
        v = torch.gather(torch.softmax(y, 1), 1, ids.long())
        return ((v / v.sum(1, keepdim=True) if normalize else v) * g.double()).sum(1)

    for e in range(10):
        h = torch.zeros(10, dtype=torch.float64, device=DEV)
        h[e] = 1e-4
        num = (f(x.double() + h) - f(x.double() - h)) / 2e-4
        # the difference's own error is h^2 / 6 times a third derivative of order 1
        assert float((num - d[:, e]).abs().max()) < 1e-6


def test_route_ties_and_zeros():
    x = torch.tensor([[0.0, -0.0, 0.0, -0.0, -1.0], [3.0, 3.0, 3.0, 3.0, 3.0], [-0.0, 0.0, 5.0, 0.0, 5.0]], device=DEV)
    for dtype in FLOATS:
        _, ids = mb.expert_route(x.to(dtype), 4)
        assert ids.tolist() == [[0, 1, 2, 3], [0, 1, 2, 3], [2, 4, 0, 1]]


@pytest.mark.parametrize("dtype", FLOATS)
def test_route_special_scores(dtype):
    low = torch.finfo(dtype).min
    x = torch.tensor([[1.0, -INF, -INF, -INF], [-INF] * 4, [low, low, 2.0, -INF], [low] * 4, [1.0, NAN, 2.0, -INF],
                      [1.0, INF, 2.0, -INF], [torch.finfo(dtype).max, 0.0, 0.0, low]], dtype=dtype, device=DEV)
    for normalize in (True, False):
        w, ids = mb.expert_route(x, 3, normalize=normalize)
        assert ids.tolist() == [[0, -1, -1], [-1, -1, -1], [2, 0, 1], [0, 1, 2], [1, 2, 0], [1, 2, 0], [0, 1, 2]]
        assert w[0].tolist() == [1, 0, 0] and w[1].tolist() == [0, 0, 0] and w[2].tolist() == [1, 0, 0]
        even = 1 / 3 if normalize else 1 / 4
        assert bool((w[3] - even).abs().max() < 4 * 2.0 ** -23)
        assert bool(w[4].isnan().all()) and bool(w[5].isnan().all()) and w[6].tolist() == [1, 0, 0]
        d = mb.expert_route_backward(torch.ones_like(w), x, ids, normalize=normalize)
        assert bool((d[:2] == 0).all()) and d.isfinite()[[0, 1, 2, 3, 6]].all()


def plain_balance(x, ids, mask):
    E = x.shape[1]
    on = torch.ones(x.shape[0], dtype=torch.bool, device=DEV) if mask is None else mask
    kept = ids[on]
    kept = kept[(kept >= 0) & (kept < E)].long()
    counts = torch.bincount(kept, minlength=E)
    n, S = int(on.sum()), int(counts.sum())
    p = softmax(x)
    slope = E * counts.double() / (S * n) if S and n else torch.zeros(E, dtype=torch.float64, device=DEV)
    d = torch.where(on[:, None], p * (slope - (p @ slope)[:, None]), 0.0)
    size = torch.where(on[:, None], p * (slope + (p @ slope)[:, None]), 0.0)
    return float(slope @ p[on].sum(0)), counts, n, d, size


@pytest.mark.parametrize("T,E,k", [(1, 1, 1), (1, 8, 2), (7, 60, 4), (100, 64, 8), (1000, 128, 8), (333, 100, 1),
                                   (5000, 8, 2), (20000, 256, 4), (90, 1024, 8), (257, 513, 3), (40, 6, 6)])
@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("pad", [0.0, 0.4])
def test_balance_and_gradient(T, E, k, dtype, pad):
    g = gen(T + E + k)
    x = (torch.randn(T, E, generator=g) * 2).to(dtype).to(DEV)
    if T > 4:
        x[3] = -INF
    ids = torch.randint(-2, E + 2, (T, k), generator=g).to(DEV)
    mask = (torch.rand(T, generator=g) >= pad).to(DEV) if pad else None
    if mask is not None and not bool(mask.all()):
        x[~mask] = NAN                       # tokens left out are not looked at
    loss, counts, n, d, size = plain_balance(x if mask is None else torch.where(mask[:, None], x, 0), ids, mask)
    for kind in (torch.int32, torch.int64):
        b = mb.expert_balance(x, ids.to(kind), mask)
        assert torch.equal(b.counts.long(), counts) and int(b.tokens) == n
        # a sum over T tokens is taken in at most T + 300 steps
        assert abs(float(b.loss) - loss) <= loss * 2.0 ** -23 * (E + T + 320)
    up = torch.tensor(0.37, device=DEV)
    got = mb.expert_balance_backward(up, x, b, mask)
    assert got.dtype is dtype
    close(got, 0.37 * d, 0.37 * size, 2 * E + 40)
    if mask is not None:
        assert bool((got[~mask] == 0).all())


def test_balance_of_nothing():
    x = torch.randn(5, 6, device=DEV)
    ids = torch.zeros(5, 2, dtype=torch.int32, device=DEV)
    none = torch.zeros(5, dtype=torch.bool, device=DEV)
    for b, m in ((mb.expert_balance(x, ids, none), none), (mb.expert_balance(x, ids - 1), None)):
        assert float(b.loss) == 0 and int(b.counts.sum()) == 0
        assert bool((mb.expert_balance_backward(torch.ones((), device=DEV), x, b, m) == 0).all())
    b = mb.expert_balance(x[:0], ids[:0])
    assert float(b.loss) == 0 and b.counts.tolist() == [0] * 6 and int(b.tokens) == 0
    assert mb.expert_balance_backward(torch.ones((), device=DEV), x[:0], b).shape == (0, 6)
    assert mb.expert_route(x[:0], 2)[0].shape == (0, 2)
    assert mb.expert_route_backward(torch.zeros(0, 2, device=DEV), x[:0], ids[:0]).shape == (0, 6)


@pytest.mark.parametrize("E,k", [(4, 4), (1, 1), (60, 60), (300, 1)])
def test_even_load_has_no_gradient(E, k):
    """The probabilities of a row sum to 1, so equal counts leave nothing of the gradient."""
    T = 3 * E
    x = (torch.randn(T, E, generator=gen(E)) * 3).to(DEV)
    ids = (torch.arange(T)[:, None] + torch.arange(k)[None]).remainder(E).to(DEV)
    b = mb.expert_balance(x, ids)
    assert b.counts.tolist() == [3 * k] * E
    assert not bool(mb.expert_balance_backward(torch.ones((), device=DEV), x, b).any())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_autograd(dtype):
    """Both losses through the graph, as a training step sums them."""
    T, E, k = 50, 24, 3
    x = (torch.randn(T, E, generator=gen(3)) * 2).to(dtype).to(DEV).requires_grad_()
    up = torch.randn(T, k, generator=gen(4)).to(DEV)
    for normalize in (True, False):
        w, ids = mb.expert_route(x, k, normalize=normalize)
        b = mb.expert_balance(x, ids)
        assert not ids.requires_grad and not b.counts.requires_grad
        (got,) = torch.autograd.grad((w * up).sum() + 0.5 * b.loss, x)
        want = mb.expert_route_backward(up, x.detach(), ids, normalize=normalize) + \
            mb.expert_balance_backward(torch.tensor(0.5, device=DEV), x.detach(), b)
        assert torch.equal(got, want)
    w, ids = mb.expert_route(x, k)
    (first,) = torch.autograd.grad(w.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        first.sum().backward()


def test_layouts_and_repeats():
    T, E, k = 90, 40, 4
    wide = torch.randn(T, E + 9, generator=gen(5)).to(DEV)
    mask = (torch.rand(2 * T, generator=gen(6)) < 0.7).to(DEV)[::2]
    for x in (wide[:, 1:E + 1], wide[:, 4:E + 4], wide.t().contiguous().t()[:, :E], wide[:1, :E].expand(T, E)):
        c = x.contiguous()
        a, b = mb.expert_route(x, k), mb.expert_route(c, k)
        assert all(torch.equal(u, v) for u, v in zip(a, b))
        p, q = mb.expert_balance(x, a[1], mask), mb.expert_balance(c, a[1], mask.contiguous())
        assert all(torch.equal(u, v) for u, v in zip(p, q))
        up = torch.randn(T, k, generator=gen(7)).to(DEV)
        assert torch.equal(mb.expert_route_backward(up, x, a[1]), mb.expert_route_backward(up, c, b[1]))
        one = torch.ones((), device=DEV)
        assert torch.equal(mb.expert_balance_backward(one, x, p, mask), mb.expert_balance_backward(one, c, q, mask))


def test_entries_named_twice():
    """The same expert twice in a row: both entries' gradients reach it."""
    x = torch.randn(4, 8, generator=gen(8)).to(DEV)
    ids = torch.tensor([[1, 1, 3], [0, 2, 0], [5, 5, 5], [7, -1, 7]], dtype=torch.int32, device=DEV)
    g = torch.randn(4, 3, generator=gen(9)).to(DEV)
    leaf = x.double().requires_grad_()
    v = torch.gather(torch.softmax(leaf, 1), 1, ids.clamp_min(0).long()) * (ids >= 0)
    for normalize in (True, False):
        w = v / v.sum(1, keepdim=True) if normalize else v
        (want,) = torch.autograd.grad((w * g.double()).sum(), leaf, retain_graph=True)
        got = mb.expert_route_backward(g, x, ids, normalize=normalize)
        assert float((got.double() - want).abs().max()) < 64 * 2.0 ** -23 * float(g.abs().max()) * 3


def test_capture():
    T, E, k = 64, 32, 4
    x = torch.randn(T, E, generator=gen(10)).to(DEV)
    up = torch.randn(T, k, generator=gen(11)).to(DEV)
    one = torch.ones((), device=DEV)

    def step():
        w, ids = mb.expert_route(x, k)
        b = mb.expert_balance(x, ids)
        return (w, ids, b.loss, b.counts, mb.expert_route_backward(up, x, ids), mb.expert_balance_backward(one, x, b))

    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    x.copy_(torch.randn(T, E, generator=gen(12)))
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(out, step()))


def test_refusals():
    x = torch.randn(4, 8, device=DEV)
    ids = torch.zeros(4, 2, dtype=torch.int32, device=DEV)
    b = mb.expert_balance(x, ids)
    one = torch.ones((), device=DEV)
    cases = [
        (lambda: mb.expert_route(x.double(), 2), NotImplementedError),
        (lambda: mb.expert_route(x, 0), ValueError), (lambda: mb.expert_route(x, 9), ValueError),
        (lambda: mb.expert_route(torch.randn(2, 1025, device=DEV), 2), ValueError),
        (lambda: mb.expert_route(torch.randn(2, 100, device=DEV), 65), ValueError),
        (lambda: mb.expert_route(x[0], 2), AssertionError),
        (lambda: mb.expert_route_backward(x[:, :2].double(), x, ids), NotImplementedError),
        (lambda: mb.expert_route_backward(x[:, :3], x, ids), AssertionError),
        (lambda: mb.expert_route_backward(x[:, :2], x, ids.float()), NotImplementedError),
        (lambda: mb.expert_balance(x, ids[:3]), AssertionError),
        (lambda: mb.expert_balance(x, ids, ids[:, 0]), NotImplementedError),
        (lambda: mb.expert_balance(x, ids, torch.ones(3, dtype=torch.bool, device=DEV)), AssertionError),
        (lambda: mb.expert_balance(x, ids.cpu()), AssertionError),
        (lambda: mb.expert_balance_backward(1.0, x, b), AssertionError),
        (lambda: mb.expert_balance_backward(one, x, b._replace(counts=b.counts[:3])), AssertionError),
    ]
    for i, (call, error) in enumerate(cases):
        with pytest.raises(error):
            call()
            pytest.fail(f"case {i} was not refused")
