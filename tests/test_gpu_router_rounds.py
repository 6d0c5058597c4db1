"""The router and its balance loss over many rows: warps take several rounds of rows, the balance several
clusters whose sums a second launch adds up.

Rows with one finite score have probabilities of exactly 0 and 1, whose sums are whole numbers: a row lost or
counted twice shows.  Bounds of the others: CUDA states 2 + floor(1.173 |y|) units in the last place for
__expf(y) and 2 for __fdividef(x, y); a unit is at most 2^-23 of the value.  y = x - max is rounded by
2^-24 |y|, which moves its exponential by |y| / 2 units.  The sum over a row is off by the mean of its terms'
errors, and the mean of |y| under the probabilities is at most their entropy, ln E; adding E terms is off
by E / 2 units.  So a probability is off by at most

    r(y) = 1.673 (|y| + ln E) + E / 2 + 10

units of 2^-23 of it, the last 10 being the two constants, the division and the products.  The weights divided by
their own sum are the same with fewer terms.  Values below 2^-126 may be 0.
"""
from __future__ import annotations

import math

import pytest
import torch

import metalblas_b200 as mb

pytestmark = pytest.mark.gpu
DEV = "cuda"
INF, NAN = math.inf, math.nan
FLOATS = (torch.float32, torch.float16, torch.bfloat16)
HALF_STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
LEAST = {torch.float32: 2.0 ** -126, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -126}
U = 2.0 ** -23


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def scores(T, E, dtype, g):
    x = torch.randn(T, E, generator=g, device=DEV) * 3
    return torch.where(torch.rand(T, E, generator=g, device=DEV) < 0.1, -INF, x).to(dtype)


def softmax(x):
    """p and r(y) in 64 bits, rows of -inf alone 0."""
    x = x.double()
    top = x.amax(1, keepdim=True)
    y = torch.where(top == -INF, -INF, x - torch.where(top == -INF, 0.0, top))
    e = y.exp()
    total = e.sum(1, keepdim=True)
    E = x.shape[1]
    r = torch.where(y > -INF, 1.673 * (y.abs() + math.log(E)) + E / 2 + 10, 0.0)
    return e / torch.where(total == 0, 1.0, total), r


# Rows of a round: 6 blocks an SM of 8 warps, 4 rows a warp up to 128 experts (28416 on 148 SMs), 2 up to 256.
@pytest.mark.parametrize("T,E,k", [(30001, 100, 8), (61000, 8, 2), (29000, 64, 4), (60000, 128, 5), (15000, 256, 8), (30000, 200, 40),
                                   (8000, 512, 4), (15001, 1000, 3)])
@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("normalize", [True, False])
def test_route_and_gradient(T, E, k, dtype, normalize):
    g = gen(T + E)
    x = scores(T, E, dtype, g)
    x[T // 3] = -INF
    grad = torch.randn(T, k, generator=g, device=DEV)
    w, ids = mb.expert_route(x, k, normalize=normalize)
    order = torch.sort(x.double(), dim=1, descending=True, stable=True).indices[:, :k]
    usable = torch.gather(x, 1, order) > -INF
    assert torch.equal(ids, torch.where(usable, order, -1).to(torch.int32))
    p, r = softmax(x)
    at = torch.where(usable, order, 0)
    want = torch.where(usable, torch.gather(p, 1, at), 0.0)
    rw = torch.where(usable, torch.gather(r, 1, at), 0.0)
    if normalize:
        total = want.sum(1, keepdim=True)
        want = want / torch.where(total == 0, 1.0, total)
    assert bool(((w.double() - want).abs() <= rw * U * want + LEAST[torch.float32]).all())

    d = mb.expert_route_backward(grad, x, ids, normalize=normalize)
    G = torch.where(usable, grad.double(), 0.0)
    mean, size = (want * G).sum(1, keepdim=True), (want * G).abs().sum(1, keepdim=True)
    worst = (want * G.abs() * rw).sum(1, keepdim=True)          # of the mean, by its terms
    put = (lambda v: torch.zeros(T, E, dtype=torch.float64, device=DEV).scatter_add(1, at, torch.where(usable, v, 0.0)))
    if normalize:
        dl, tol = put(want * (G - mean)), put(want * ((G.abs() + size) * (rw + E / 2 + 10) + worst))
    else:
        dl, tol = put(want * G) - p * mean, put(want * G.abs() * (rw + 10)) + p * (size * (r + E / 2 + 10) + worst)
    assert d.dtype is dtype
    tol = U * tol * (1 + HALF_STEP[dtype]) + HALF_STEP[dtype] * dl.abs() + LEAST[dtype]
    err = (d.double() - dl).abs()
    assert bool((err <= tol).all()), float((err / tol).max())


@pytest.mark.parametrize("T,E,k", [(700, 8, 2), (5000, 64, 4), (20000, 100, 2), (20000, 256, 3), (3000, 1000, 2), (100003, 8, 1), (2049, 513, 2),
                                   (513, 128, 1), (260, 512, 1)])
@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("masked", [False, True])
def test_every_row_counts_once(T, E, k, dtype, masked):
    """One-hot rows: loss E sum_e c_e s_e / (S n) of whole numbers c (entries) and s (rows); its E products
    and sums and one rounding are off by E + 12 units of 2^-24 and the probability of 1, an inverse of 1, by 4,
    a row more or less by about 1 / T."""
    g = gen(T + E + k)
    hot = torch.randint(0, E, (T,), generator=g, device=DEV)
    x = torch.full((T, E), -INF, dtype=dtype, device=DEV)
    x.scatter_(1, hot[:, None], torch.randn(T, 1, generator=g, device=DEV).to(dtype))
    ids = torch.randint(0, E, (T, k), generator=g, device=DEV).to(torch.int32)
    mask = torch.rand(T, generator=g, device=DEV) < 0.7 if masked else None
    on = torch.ones(T, dtype=torch.bool, device=DEV) if mask is None else mask
    x[~on] = NAN
    b = mb.expert_balance(x, ids, mask)
    c, s = torch.bincount(ids[on].flatten(), minlength=E), torch.bincount(hot[on], minlength=E)
    n, S = int(on.sum()), int(c.sum())
    assert torch.equal(b.counts.long(), c) and int(b.tokens) == n
    want = E * int((c * s).sum()) / (S * n)
    tol = (E + 16) * 2.0 ** -24
    least = int(c[c > 0].min()) / int((c * s).sum())         # what one row of the least loaded expert adds
    assert abs(float(b.loss) - want) <= tol * want
    if E <= 256 and T > 1000:
        assert tol < least, "the bound would not show a lost row"
    # p = 1 times (a - a): no row has a gradient but what that p's 4 units of 2^-24 leave
    d = mb.expert_balance_backward(torch.ones((), device=DEV), x, b, mask)
    assert not bool(d[~on].any())
    assert float(d.abs().max()) <= 4 * 2.0 ** -24 * float((E * c - S).abs().max()) / (S * n) * 1.01


@pytest.mark.parametrize("T,E,k", [(30001, 100, 8), (100003, 8, 2), (70000, 64, 4), (15000, 256, 8), (9000, 1000, 3)])
@pytest.mark.parametrize("dtype", FLOATS)
def test_balance_and_gradient(T, E, k, dtype):
    """The loss by the depth of its sum: a lane's rows, 8 warps, 8 blocks and at most 74 clusters one after
    another, E products."""
    g = gen(T * 3 + E)
    x = scores(T, E, dtype, g)
    mask = torch.rand(T, generator=g, device=DEV) < 0.8
    x[~mask] = NAN
    ids = torch.randint(-1, E + 1, (T, k), generator=g, device=DEV)
    b = mb.expert_balance(x, ids, mask)
    kept = ids[mask]
    c = torch.bincount(kept[(kept >= 0) & (kept < E)], minlength=E)
    n, S = int(mask.sum()), int(c.sum())
    assert torch.equal(b.counts.long(), c) and int(b.tokens) == n
    p, r = softmax(torch.where(mask[:, None], x, -INF))
    slope = E * c.double() / (S * n)
    want = float(slope @ p.sum(0))
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    lanes = min(T, sms * 4 // 8 * 8 * 8)                      # warps of all clusters
    depth = math.ceil(T / lanes) + 4 + 8 + 8 + sms * 4 // 8 + E + 12
    tol = U * (float(slope @ (p * r).sum(0)) + depth / 2 * want)
    assert abs(float(b.loss) - want) <= tol, (abs(float(b.loss) - want) / tol, tol / want)

    got = mb.expert_balance_backward(torch.tensor(0.73, device=DEV), x, b, mask)
    # a less its mean, as the kernel takes it: E c - S whole numbers, one rounding, times a factor of two roundings
    a = float(torch.tensor(0.73)) * (slope - slope.mean())
    mean, size = (p @ a)[:, None], (p @ a.abs())[:, None]
    worst = ((p * r) @ a.abs())[:, None]
    dl = torch.where(mask[:, None], p * (a - mean), 0.0)
    tol = U * p * ((a.abs() + size) * (r + E / 2 + 10) + worst) * (1 + HALF_STEP[dtype]) + HALF_STEP[dtype] * dl.abs() + LEAST[dtype]
    err = (got.double() - dl).abs()
    assert bool((err <= tol).all()), float((err / tol).max())
