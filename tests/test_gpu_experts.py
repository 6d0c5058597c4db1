"""Tokens sorted by expert and back, against the formulas: whole numbers equal, sums within
the roundings of an fp32 sum of their length and one rounding to the type."""
from __future__ import annotations

import pytest
import torch

import metalblas_b200 as mb

pytestmark = pytest.mark.gpu
DEV = "cuda"
FLOATS = (torch.float32, torch.float16, torch.bfloat16)
U32 = 2.0 ** -24
UNIT = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -24, torch.bfloat16: 2.0 ** -133}


def gen(seed):
    return torch.Generator().manual_seed(seed)


def route(T, k, E, g, drop=0.0, dtype=torch.int64):
    ids = torch.stack([torch.randperm(E, generator=g)[:k] for _ in range(T)]) if T and k <= E else \
        torch.randint(0, E, (T, k), generator=g)
    ids = torch.where(torch.rand(T, k, generator=g) < drop, torch.tensor(-1), ids)
    return ids.to(dtype).to(DEV)


def plain_sort(ids, E):
    flat = ids.reshape(-1).cpu().tolist()
    key = [e if 0 <= e < E else E for e in flat]
    order = sorted(range(len(flat)), key=lambda i: key[i])
    position = [0] * len(flat)
    for s, i in enumerate(order):
        position[i] = s
    return order, position, [sum(x < e for x in key) for e in range(E + 1)]


SORTS = [(1, 1, 1), (1, 2, 8), (3, 1, 4), (16, 2, 8), (33, 4, 60), (100, 8, 64), (257, 3, 128), (5, 8, 1024),
         (1000, 2, 7), (4097, 1, 256), (3000, 8, 512), (20000, 4, 16), (40000, 4, 70)]


@pytest.mark.parametrize("T,k,E", SORTS)
@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
def test_sort(T, k, E, dtype):
    ids = route(T, k, E, gen(T + E), drop=0.2, dtype=dtype)
    got = mb.expert_sort(ids, E)
    order, position, offsets = plain_sort(ids, E)
    assert got.order.tolist() == order
    assert got.position.reshape(-1).tolist() == position and got.position.shape == ids.shape
    assert got.offsets.tolist() == offsets


@pytest.mark.parametrize("what", ["one expert", "all dropped", "last only", "out of range", "large numbers"])
def test_sort_uneven(what):
    T, k, E = 700, 2, 9
    ids = route(T, k, E, gen(1))
    if what == "one expert":
        ids = torch.full_like(ids, 4)
    elif what == "all dropped":
        ids = torch.full_like(ids, -1)
    elif what == "last only":
        ids = torch.where(torch.arange(T, device=DEV)[:, None] % 3 == 0, E - 1, -5)
        ids = ids.expand(T, k)
    elif what == "out of range":
        ids = ids + 3
    else:
        ids = torch.where(ids == 2, 2 + (1 << 32), ids)  # 2 in the low 32 bits only
    got = mb.expert_sort(ids, E)
    order, position, offsets = plain_sort(ids, E)
    assert got.order.tolist() == order and got.offsets.tolist() == offsets
    assert got.position.reshape(-1).tolist() == position


def test_sort_empty_and_strided():
    got = mb.expert_sort(torch.zeros(0, 2, dtype=torch.int64, device=DEV), 3)
    assert got.order.numel() == 0 and got.offsets.tolist() == [0, 0, 0, 0]
    ids = route(40, 6, 8, gen(2))
    a, b = mb.expert_sort(ids[:, ::2], 8), mb.expert_sort(ids[:, ::2].contiguous(), 8)
    assert all(torch.equal(x, y) for x, y in zip(a, b))


def close(got, want, size, terms):
    """|got - want| within `terms` fp32 roundings of `size` and one rounding of the type."""
    u = UNIT[got.dtype]
    tol = terms * U32 * size * (1 + u) + u * want.abs() + TINY[got.dtype]
    assert bool(((got.double() - want).abs() <= tol).all())


def taken(rows, o):
    """The rows of each entry in 64 bits, zero for dropped ones."""
    kept = o.position < o.offsets[-1]
    return torch.where(kept[..., None], rows.double()[o.position.long()], 0.0)


CASES = [(1, 1, 1, 1), (1, 2, 8, 64), (3, 2, 4, 7), (16, 2, 8, 4096), (33, 8, 60, 130), (40, 9, 16, 264),
         (257, 3, 128, 1000), (64, 1, 4, 8192), (7, 17, 20, 48), (500, 4, 8, 515)]


@pytest.mark.parametrize("T,k,E,H", CASES)
@pytest.mark.parametrize("dtype", FLOATS)
def test_gather_combine_and_gradients(T, k, E, H, dtype):
    g = gen(T + k + E + H)
    o = mb.expert_sort(route(T, k, E, g, drop=0.25), E)
    x = torch.randn(T, H, generator=g).to(dtype).to(DEV)
    kept = int(o.offsets[-1])
    xs = mb.expert_gather(x, o)
    assert torch.equal(xs[:kept], x[(o.order[:kept] // k).long()]) and bool((xs[kept:] == 0).all())
    q, s = mb.expert_gather_quantize(x, o)
    wq, ws = mb.quantize(xs)
    assert torch.equal(q, wq) and torch.equal(s, ws)
    y = torch.randn(T * k, H, generator=g).to(dtype).to(DEV)
    d = torch.randn(T, H, generator=g).to(dtype).to(DEV)
    for wdt in {dtype, torch.float32}:
        w = torch.rand(T, k, generator=g).to(wdt).to(DEV)
        yt, wd = taken(y, o), w.double()[..., None]
        close(mb.expert_combine(y, w, o), (yt * wd).sum(1), (yt * wd).abs().sum(1), k + 1)
        dy, dw = mb.expert_combine_backward(d, y, w, o)
        want = torch.zeros_like(y).double()
        live = (o.position < o.offsets[-1])[..., None]
        want[o.position.long()] = torch.where(live, wd * d.double()[:, None], 0.0)
        close(dy, want, want.abs(), 1)
        p = yt * d.double()[:, None]
        assert dw.dtype is wdt
        close(dw, p.sum(-1), p.abs().sum(-1), H + 1)
    ones = taken(y, o)
    close(mb.expert_gather_backward(y, o), ones.sum(1), ones.abs().sum(1), k + 1)


@pytest.mark.parametrize("dtype", FLOATS)
def test_rows_of_dropped_entries_are_never_read(dtype):
    """NaN and infinity in the rows past the kept ones reach no result."""
    g = gen(31)
    T, k, E, H = 20, 3, 5, 72
    ids = route(T, k, E, g, drop=0.4)
    ids[4] = -1   # a token with no expert at all
    o = mb.expert_sort(ids, E)
    kept = int(o.offsets[-1])
    y = torch.randn(T * k, H, generator=g).to(dtype).to(DEV)
    y[kept:] = float("nan")
    y[kept::2] = float("inf")
    w = torch.rand(T, k, generator=g).to(DEV)
    clean = y.clone()
    clean[kept:] = 0
    d = torch.randn(T, H, generator=g).to(dtype).to(DEV)
    out = mb.expert_combine(y, w, o)
    assert torch.equal(out, mb.expert_combine(clean, w, o)) and bool((out[4] == 0).all())
    for a, b in zip(mb.expert_combine_backward(d, y, w, o), mb.expert_combine_backward(d, clean, w, o)):
        assert torch.equal(a, b)
    assert bool((mb.expert_combine_backward(d, y, w, o)[1][4] == 0).all())
    assert torch.equal(mb.expert_gather_backward(y, o), mb.expert_gather_backward(clean, o))


def test_gradients_against_differences():
    """combine is linear in rows and in weights, so its differences along a direction are its
    derivative: <gradient, direction> equals them up to the gradients' own roundings."""
    g = gen(32)
    T, k, E, H = 30, 3, 6, 50
    o = mb.expert_sort(route(T, k, E, g, drop=0.2), E)
    y, w = torch.randn(T * k, H, generator=g).to(DEV), torch.rand(T, k, generator=g).to(DEV)
    d, u = torch.randn(T, H, generator=g).to(DEV), torch.randn(T * k, H, generator=g).to(DEV)
    v, x = torch.randn(T, k, generator=g).to(DEV), torch.randn(T, H, generator=g).to(DEV)

    def loss(yy, ww):
        return float(((taken(yy, o) * ww.double()[..., None]).sum(1) * d.double()).sum())

    dy, dw = mb.expert_combine_backward(d, y, w, o)
    for grad, along, size, diff in (
            (dy, u, (dy.double() * u.double()).abs().sum(),
             (loss(y.double() + u.double(), w) - loss(y.double() - u.double(), w)) / 2),
            (dw, v, (taken(y, o) * d.double()[:, None] * v.double()[..., None]).abs().sum() * H,
             (loss(y, w.double() + v.double()) - loss(y, w.double() - v.double())) / 2)):
        assert abs(float((grad.double() * along.double()).sum()) - diff) <= 2 * U32 * float(size)
    kept = int(o.offsets[-1])

    def gathered(xx):
        return float((xx.double()[(o.order[:kept] // k).long()] * u[:kept].double()).sum())

    dx = mb.expert_gather_backward(u, o)
    diff = (gathered(x.double() * 2) - gathered(x.double() * 0)) / 2
    size = float((taken(u, o).abs().sum(1) * x.double().abs()).sum())
    assert abs(float((dx.double() * x.double()).sum()) - diff) <= (k + 1) * U32 * size


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_autograd_is_the_gradients(dtype):
    g = gen(33)
    T, k, E, H = 25, 2, 4, 96
    ids = route(T, k, E, g, drop=0.1)
    x = torch.randn(T, H, generator=g).to(dtype).to(DEV).requires_grad_()
    w = torch.rand(T, k, generator=g).to(DEV).requires_grad_()
    o = mb.expert_sort(ids, E)
    xs = mb.expert_gather(x, o)
    out = mb.expert_combine(xs * 2, w, o)
    d = torch.randn(T, H, generator=g).to(dtype).to(DEV)
    out.backward(d)
    dy, dw = mb.expert_combine_backward(d, (xs * 2).detach(), w.detach(), o)
    assert torch.equal(w.grad, dw)
    assert torch.equal(x.grad, mb.expert_gather_backward(dy * 2, o))
    rows = torch.randn(T * k, H, generator=g).to(dtype).to(DEV).requires_grad_()
    mb.expert_combine(rows, None, o).backward(d)
    assert torch.equal(rows.grad, mb.expert_combine_backward(d, rows.detach(), torch.ones(T, k, device=DEV), o)[0])
    with torch.no_grad():
        assert not mb.expert_gather(x, o).requires_grad


def test_layouts_and_repeats():
    g = gen(34)
    T, k, E, H = 50, 4, 8, 200
    o = mb.expert_sort(route(T, k, E, g, drop=0.1), E)
    big = torch.randn(2 * T, 2 * H + 3, generator=g).to(torch.bfloat16).to(DEV)
    rows = torch.randn(T * k, 2 * H + 3, generator=g).to(torch.bfloat16).to(DEV)
    w = torch.rand(k, T, generator=g).to(DEV).t()
    for c in (slice(0, H), slice(1, H + 1), slice(3, H + 2), slice(0, 2 * H, 2)):
        x, y, d = big[::2, c], rows[:, c], big[1::2, c]
        assert torch.equal(mb.expert_gather(x, o), mb.expert_gather(x.contiguous(), o))
        a, b = mb.expert_gather_quantize(x, o), mb.expert_gather_quantize(x.contiguous(), o)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
        assert torch.equal(mb.expert_combine(y, w, o), mb.expert_combine(y.contiguous(), w.contiguous(), o))
        p, q = mb.expert_combine_backward(d, y, w, o), mb.expert_combine_backward(d.contiguous(), y.contiguous(),
                                                                                 w.contiguous(), o)
        assert torch.equal(p[0], q[0])
        again = mb.expert_combine_backward(d, y, w, o)
        assert torch.equal(p[0], again[0]) and torch.equal(p[1], again[1])
    row = big[:1, :H].expand(T, H)   # one row for every token
    assert torch.equal(mb.expert_gather(row, o), mb.expert_gather(row.contiguous(), o))


def test_slots_outside_the_buffer_are_skipped():
    """A position that is no slot reads and writes nothing."""
    g = gen(35)
    T, k, H = 6, 2, 64
    pos = torch.arange(T * k, dtype=torch.int32).reshape(T, k)
    pos[1, 0], pos[2, 1] = -7, 1 << 30
    off = torch.tensor([0, 1 << 30], dtype=torch.int32)
    o = mb.ExpertOrder(None, pos.to(DEV), off.to(DEV))
    x, y = torch.randn(T, H, generator=g).to(DEV), torch.randn(T * k, H, generator=g).to(DEV)
    w = torch.ones(T, k, device=DEV)
    out = mb.expert_combine(y, w, o)
    want = y.view(T, k, H).clone()
    want[1, 0] = 0
    want[2, 1] = 0
    assert torch.equal(out, want.sum(1))
    xs = mb.expert_gather(x, o).view(T, k, H)
    assert torch.equal(xs[0], x[0].expand(k, H)) and torch.equal(xs[1, 1], x[1])
    assert float(mb.expert_combine_backward(x, y, w, o)[1][1, 0]) == 0


def test_a_layer_runs_together():
    """Sort, gather with quantization, experts' int8 products, combine: against the layer in
    64 bits on the quantized operands."""
    g = gen(36)
    T, k, E, K, N = 90, 2, 6, 256, 144
    ids = route(T, k, E, g, drop=0.1)
    x = torch.randn(T, K, generator=g).to(torch.bfloat16).to(DEV)
    wf = (0.02 * torch.randn(E, N, K, generator=g)).to(DEV)
    wq, sw = mb.quantize(wf)
    weights = torch.rand(T, k, generator=g).to(DEV)
    o = mb.expert_sort(ids, E)
    q, s = mb.expert_gather_quantize(x, o)
    y = mb.grouped_scaled_mm(q, wq.transpose(1, 2), s, sw, o.offsets, out_dtype=torch.float32)
    out = mb.expert_combine(y, weights, o)
    qx, sx = mb.quantize(x)
    deq = qx.double() * sx.double()[:, None]
    want, size = torch.zeros(T, N, dtype=torch.float64, device=DEV), torch.zeros(T, N, dtype=torch.float64, device=DEV)
    for t in range(T):
        for j in range(k):
            e = int(ids[t, j])
            if e >= 0:
                v = (deq[t] @ (wq[e].double() * sw[e].double()[:, None]).t()) * weights[t, j].double()
                want[t] += v
                size[t] += v.abs()
    close(out, want, size, 4 + k + 1)


def test_refusals():
    z = lambda *s, dt=torch.int64: torch.zeros(*s, dtype=dt, device=DEV)  # noqa: E731
    f = lambda *s, dt=torch.float32: torch.ones(*s, dtype=dt, device=DEV)  # noqa: E731
    with pytest.raises(AssertionError):
        mb.expert_sort(torch.zeros(2, 2, dtype=torch.int64), 4)
    with pytest.raises(AssertionError):
        mb.expert_sort(z(4), 4)
    with pytest.raises(NotImplementedError):
        mb.expert_sort(z(4, 2, dt=torch.int16), 4)
    for E in (0, 1025):
        with pytest.raises(ValueError):
            mb.expert_sort(z(4, 2), E)
    o = mb.expert_sort(z(4, 2), 3)
    with pytest.raises(AssertionError):
        mb.expert_gather(f(5, 8), o)
    with pytest.raises(NotImplementedError):
        mb.expert_gather(f(4, 8, dt=torch.float64), o)
    with pytest.raises(AssertionError):
        mb.expert_gather(f(4, 8).cpu(), o)
    with pytest.raises(NotImplementedError):
        mb.expert_gather(f(4, 8), o._replace(position=o.position.long()))
    with pytest.raises(AssertionError):
        mb.expert_combine(f(7, 8), f(4, 2), o)
    with pytest.raises(AssertionError):
        mb.expert_combine(f(8, 8), f(2, 4), o)
    with pytest.raises(NotImplementedError):
        mb.expert_combine(f(8, 8), f(4, 2, dt=torch.float16), o)
    with pytest.raises(NotImplementedError):
        mb.expert_combine_backward(f(4, 8, dt=torch.float16), f(8, 8), f(4, 2), o)
    with pytest.raises(AssertionError):
        mb.expert_combine_backward(f(4, 9), f(8, 8), f(4, 2), o)
