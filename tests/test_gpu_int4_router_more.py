"""4-bit products and the router where the plain tests do not go: every kernel and tile by force,
the host fast path against the Python path, operands past 2^31 elements, threads and streams,
broadcast weights, and operands that want a gradient.

The exact inputs of tests/test_gpu_int4.py make a product the exact value rounded once in any
order of summing, so every plan has to give the same bits."""
from __future__ import annotations

import threading

import pytest
import torch
import torch.autograd.forward_ad as fwd

import metalblas_b200 as mb
from metalblas_b200 import _lib, int4, kernels, router
from tests.test_gpu_int4 import DEV, TOKENS, close, gen, split, tokens, unpacked, weights

pytestmark = pytest.mark.gpu
PLANS = [(1, 0), (2, 0)] + [(bn, sp) for bn in (16, 32, 64, 128) for sp in (1, 2, 4, 8)] + [(256, 1)]


@pytest.fixture(autouse=True)
def alone():
    yield
    assert kernels.device_status() == 0


def by_plan(call, plan):
    try:
        return call((*plan, 0, 0))
    except ValueError as e:          # a split that K has no columns for
        assert "no kernel has plan" in str(e)


@pytest.mark.parametrize("dtype", TOKENS)
@pytest.mark.parametrize("zero", [False, True])
@pytest.mark.parametrize("M,K,N,G", [(1, 2048, 300, 128), (5, 4100, 259, 32), (19, 1031, 130, 64), (70, 2304, 513, 256),
                                     (300, 520, 264, 128), (257, 8192, 40, 64), (2, 30, 7, 32)])
def test_every_plan(M, K, N, G, dtype, zero):
    g = gen(M + K + N)
    q, s, z = weights((N,), K, G, g, dtype, zero, True)
    x = tokens(M, K, g, dtype, True)
    want = (x.double() @ unpacked(q, s, z, K, G).t()).to(dtype)
    ran = 0
    for plan in PLANS:
        got = by_plan(lambda p: mb.int4_mm(x, q, s, G, zero=z, _plan=p), plan)
        if got is not None:
            ran += 1
            assert torch.equal(got, want), plan
    assert ran >= (6 if K < 256 else 11)


@pytest.mark.parametrize("zero", [False, True])
@pytest.mark.parametrize("counts,rest,K,N,G", [([3, 0, 1, 8, 0, 40], 5, 2048, 200, 128), ([0, 0, 7], 0, 1100, 129, 32),
                                               ([200, 1, 130], 2, 768, 300, 64), ([1] * 300 + [0] * 724, 3, 256, 32, 256)])
def test_every_plan_by_group(counts, rest, K, N, G, zero):
    g = gen(sum(counts) + K)
    E, M, dtype = len(counts), sum(counts) + rest, torch.bfloat16
    q, s, z = weights((E, N), K, G, g, torch.float32, zero, True)
    x = tokens(M, K, g, dtype, True)
    off, w = split(counts), unpacked(q, s, z, K, G)
    want = torch.zeros(M, N, dtype=torch.float64, device=DEV)
    at = 0
    for e, c in enumerate(counts):
        want[at:at + c] = x[at:at + c].double() @ w[e].t()
        at += c
    for plan in PLANS:
        got = by_plan(lambda p: mb.grouped_int4_mm(x, q, s, off, G, zero=z, _plan=p), plan)
        if got is not None:
            assert torch.equal(got, want.to(dtype)), plan


def test_no_such_plan():
    q, s, _ = weights((8,), 64, 32, gen(0), torch.float32, False)
    x = tokens(2, 64, gen(1), torch.float16)
    for plan in ((3, 0), (16, 3), (256, 2), (1, 2), (16, 8)):
        with pytest.raises(ValueError):
            mb.int4_mm(x, q, s, 32, _plan=(*plan, 0, 0))


@pytest.mark.parametrize("M", [2, 90])
def test_broadcast_and_single(M):
    """One matrix for all groups (stride 0), one group whose stride is odd, one weight row, and zero
    points past 15."""
    g = gen(M)
    K, N, G = 300, 72, 64
    q, s, _ = weights((N,), K, G, g, torch.bfloat16, False, True)
    z = torch.randint(0, 256, s.shape, generator=g).to(torch.uint8).to(DEV)
    x = tokens(M, K, g, torch.bfloat16, True)
    for zero in (None, z):
        want = (x.double() @ unpacked(q, s, zero, K, G).t()).bfloat16()
        assert torch.equal(mb.int4_mm(x, q, s, G, zero=zero), want)
        off = split([M // 2, 0, M - M // 2])
        e = (lambda t: None if t is None else t.expand(3, *t.shape))
        assert torch.equal(mb.grouped_int4_mm(x, e(q), e(s), off, G, zero=e(zero)), want)
        odd = torch.empty(1, N * q.stride(0) + 17, dtype=torch.uint8, device=DEV)[:, :N * q.stride(0)]
        odd = odd.view(1, N, q.stride(0))[..., :q.shape[1]].copy_(q)
        one = (lambda t: None if t is None else t[None])
        assert torch.equal(mb.grouped_int4_mm(x, odd, s[None], split([M]), G, zero=one(zero)), want)
        assert torch.equal(mb.int4_mm(x, q[:1], s[:1], G, zero=None if zero is None else zero[:1]), want[:, :1])


def equal(a, b):
    return len(a) == len(b) and all(torch.equal(x, y) for x, y in zip(a, b))


def test_plain_calls_are_served():
    """The host fast path takes the plain call and gives the Python path's result."""
    fast = _lib.fast()
    assert fast is not None
    g = gen(3)
    w = torch.randn(48, 100, generator=g).to(DEV)
    qs = fast.try_int4_quantize(w, 32, torch.float16)
    assert qs is not None and equal(qs, int4._quantize(w, 32, torch.float16)) and qs[0].stride(0) == 64
    back = fast.try_int4_dequantize(*qs, None, 100, 32, torch.bfloat16)
    assert back is not None and torch.equal(back, int4._dequantize(*qs, 32, None, 100, torch.bfloat16))
    x, bias = tokens(5, 100, g, torch.float16), torch.randn(48, generator=g).to(DEV)
    y = fast.try_int4(x, *qs, None, 32, None, bias)
    assert y is not None and torch.equal(y, int4._int4_mm(x, *qs, 32, None, bias, None, None))
    q3, s3, z3 = weights((3, 48), 100, 32, g, torch.float32, True)
    off = split([2, 0, 3])
    y = fast.try_int4(x, q3, s3, z3, 32, off, None)
    assert y is not None and torch.equal(y, int4._grouped_int4_mm(x, q3, s3, off, 32, z3, None, None))
    logits = torch.randn(40, 12, generator=g).to(DEV)
    wi = fast.try_route(logits, 3, False)
    assert wi is not None and equal(wi, router._route(logits, 3, False))
    up, mask = torch.randn(40, 3, generator=g).to(DEV), (torch.rand(40, generator=g) < 0.8).to(DEV)
    d = fast.try_route_backward(logits, up, wi[1], False)
    assert d is not None and torch.equal(d, router._route_backward(logits, up, wi[1], False))
    b = fast.try_balance(logits, wi[1], mask)
    assert b is not None and equal(b, router._balance(logits, wi[1], mask))
    one = torch.ones((), device=DEV)
    d = fast.try_balance_backward(logits, one, b[1], b[2], mask)
    assert d is not None and torch.equal(d, router._balance_backward(logits, one, mb.ExpertBalance(*b), mask))
    # what it does not take
    leaf = logits.clone().requires_grad_()
    assert fast.try_route(leaf, 3, True) is None and fast.try_balance(leaf, wi[1], None) is None
    assert fast.try_route(logits, 13, True) is None and fast.try_balance(logits, wi[1].long(), None) is None
    assert fast.try_int4(x.float(), *qs, None, 32, None, None) is None and fast.try_int4(x, *qs, None, 48, None, None) is None
    assert fast.try_int4_quantize(w.double(), 32, torch.float16) is None and fast.try_route([1.0], 1, True) is None


def test_operands_that_want_a_derivative():
    q, s, _ = weights((16,), 64, 32, gen(0), torch.float32, False)
    x, bias = tokens(3, 64, gen(1), torch.bfloat16), torch.zeros(16, device=DEV)
    leaf = (lambda t: t.clone().requires_grad_())
    calls = [lambda f: mb.int4_mm(f(x), q, s, 32), lambda f: mb.int4_mm(x, q, f(s), 32),
             lambda f: mb.int4_mm(x, q, s, 32, bias=f(bias)), lambda f: mb.grouped_int4_mm(f(x), q[None], s[None], split([3]), 32),
             lambda f: mb.grouped_int4_mm(x, q[None], f(s)[None], split([3]), 32)]
    for call in calls:
        with pytest.raises(NotImplementedError, match="no gradient"):
            call(leaf)
        with torch.no_grad():
            assert not call(leaf).requires_grad
        with fwd.dual_level(), pytest.raises(NotImplementedError, match="forward-mode"):
            call(lambda t: fwd.make_dual(t, torch.ones_like(t)))
    logits, ids = torch.randn(3, 4, device=DEV), torch.zeros(3, 1, dtype=torch.int32, device=DEV)
    for call in (lambda t: mb.expert_route(t, 2), lambda t: mb.expert_balance(t, ids)):
        with fwd.dual_level(), pytest.raises(NotImplementedError):
            call(fwd.make_dual(logits, torch.ones_like(logits)))


def test_threads_and_streams():
    """Calls at the same time from threads on streams of their own."""
    g = gen(9)
    q, s, _ = weights((1000,), 1024, 128, g, torch.bfloat16, False)
    inputs = [(tokens(m, 1030, g, torch.bfloat16)[:, 1:1025], torch.randn(m * 40, 32, generator=g).to(DEV)) for m in (1, 7, 33, 200)]

    def work(x, logits):
        w, ids = mb.expert_route(logits, 4)
        return mb.int4_mm(x, q, s, 128), w, ids, mb.expert_balance(logits, ids).loss

    want = [work(*i) for i in inputs]
    torch.cuda.synchronize()
    got, errors = [None] * len(inputs), []

    def run(i):
        try:
            st = torch.cuda.Stream()
            with torch.cuda.stream(st):
                for _ in range(20):
                    got[i] = work(*inputs[i])
            st.synchronize()
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=run, args=(i,)) for i in range(len(inputs))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors and all(equal(a, b) for a, b in zip(want, got))


# ------------------------------------------------------------------------------ past 2^31
def test_large_weights_by_group():
    g = torch.Generator(device=DEV).manual_seed(1)
    E, N, K, G = 140, 8192, 8192, 128
    q = torch.randint(0, 256, (E, N, K // 2), dtype=torch.uint8, generator=g, device=DEV)
    assert q.numel() > 1 << 32
    s = torch.rand((E, N, K // G), generator=g, device=DEV) * 0.02 + 0.002
    for each in (1, 40):
        counts = [0] * E
        for e in (0, 64, 131, E - 1):
            counts[e] = each
        x = torch.randn(4 * each, K, generator=g, device=DEV).bfloat16()
        got = mb.grouped_int4_mm(x, q, s, split(counts), G)
        for i, e in enumerate((0, 64, 131, E - 1)):
            w, xe = unpacked(q[e, -200:], s[e, -200:], None, K, G), x[i * each:(i + 1) * each].double()
            close(got[i * each:(i + 1) * each, -200:], xe @ w.t(), xe.abs() @ w.abs().t(), K + 2 * (K // G))
    del q, s
    torch.cuda.empty_cache()


def test_large_rows_and_results():
    g = gen(2)
    M, N, K, G = 70000, 32768, 64, 32
    assert M * N > 1 << 31
    q, s, _ = weights((N,), K, G, g, torch.float32, False, True)
    wide = torch.empty(M, 32000, dtype=torch.bfloat16, device=DEV)
    assert wide.numel() > 1 << 31
    x = wide[:, 512:512 + K].copy_(tokens(M, K, g, torch.bfloat16, True))
    w = unpacked(q, s, None, K, G)
    for plan in (None, (1, 0, 0, 0)):
        y = mb.int4_mm(x, q, s, G, _plan=plan)
        for rows in (slice(0, 40), slice(M - 300, M)):
            assert torch.equal(y[rows], (x[rows].double() @ w.t()).bfloat16())
        del y
    # rows past the groups are set to zeros, far behind
    y = mb.grouped_int4_mm(x, q[None], s[None], split([10]), G)
    assert torch.equal(y[:10], (x[:10].double() @ w.t()).bfloat16()) and not bool(y[10:].any())
    del y, x
    torch.cuda.empty_cache()
    # quantize and back: a row's result does not depend on where it lies
    v = wide.normal_(generator=torch.Generator(device=DEV).manual_seed(3))
    qa, sa = mb.quantize_int4(v, 128)
    assert qa.numel() > 1 << 30
    back = mb.dequantize_int4(qa, sa, 128)
    tail = mb.quantize_int4(v[-3:].contiguous(), 128)
    assert torch.equal(qa[-3:], tail[0]) and torch.equal(sa[-3:], tail[1])
    assert torch.equal(back[-3:], mb.dequantize_int4(*tail, 128))
    del back, qa, sa, v, wide
    torch.cuda.empty_cache()


def test_large_scores():
    T, E, k = 2_200_000, 1024, 2
    x = torch.empty(T, E, dtype=torch.bfloat16, device=DEV).normal_(generator=torch.Generator(device=DEV).manual_seed(4))
    assert x.numel() > 1 << 31
    w, ids = mb.expert_route(x, k)
    up = torch.randn(T, k, device=DEV)
    d = mb.expert_route_backward(up, x, ids)
    tail = x[-5:].contiguous()
    small = mb.expert_route(tail, k)
    assert torch.equal(w[-5:], small[0]) and torch.equal(ids[-5:], small[1])
    assert torch.equal(d[-5:], mb.expert_route_backward(up[-5:], tail, small[1]))
    del d
    b = mb.expert_balance(x, ids)
    assert int(b.tokens) == T and torch.equal(b.counts.long(), torch.bincount(ids.flatten(), minlength=E))
    p = sum(torch.softmax(part.double(), 1).sum(0) for part in x.split(100000))
    want = float(E * (b.counts.double() / (T * k) * p / T).sum())
    # a lane sums some thousand rows, 8 warps, 8 blocks and 74 clusters: fewer than 2000 steps
    assert abs(float(b.loss) - want) <= want * 2.0 ** -23 * (E + 2000)
    d = mb.expert_balance_backward(torch.ones((), device=DEV), x, b)
    assert torch.equal(d[-5:], mb.expert_balance_backward(torch.ones((), device=DEV), tail, b))
    del d, x
    torch.cuda.empty_cache()


@pytest.mark.parametrize("E,counts,K,N", [(256, 4, 3743, 464), (256, 5, 4096, 464), (128, 9, 2048, 1000), (1, 8, 4096, 14336)])
@pytest.mark.parametrize("G", [32, 128, 256])
def test_weights_stream_in_order(E, counts, K, N, G):
    """Many items through each warp's ring, again and again: a copy must not overtake the reads of
    what lies there."""
    g = gen(E + K + G)
    q, s, _ = weights((E, N), K, G, g, torch.bfloat16, False, True)
    x = tokens(E * counts, K, g, torch.bfloat16, True)
    off = split([counts] * E)
    want = torch.cat([(x[e * counts:(e + 1) * counts].double() @ unpacked(q[e], s[e], None, K, G).t()).bfloat16()
                      for e in range(E)])
    for plan in ((1, 0, 0, 0), (2, 0, 0, 0), (16, 1, 0, 0), (32, 2, 0, 0)):
        for _ in range(10):
            assert torch.equal(mb.grouped_int4_mm(x, q, s, off, G, _plan=plan), want), plan
