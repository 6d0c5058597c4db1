"""Chains of kernels over one buffer whose contents change in every round.

Each kernel of a chain may start while the one before it finishes, so a buffer is read, written
again and read again by kernels that are on the device together.  The chain runs without a host
synchronisation, and every round's result is compared with the same calls run one by one.
"""
from __future__ import annotations

import pytest
import torch

import metalblas_b200 as mb
from metalblas_b200 import kernels

pytestmark = pytest.mark.gpu
DEV = "cuda"
ROUNDS = 60


@pytest.fixture(autouse=True)
def no_wait_gave_up():
    yield
    assert kernels.device_status() == 0


def gen(seed):
    return torch.Generator().manual_seed(seed)


def ints(shape, g):
    return torch.randint(-127, 128, shape, dtype=torch.int8, generator=g).to(DEV)


def scales(shape, g):
    return (torch.rand(shape, generator=g) * 0.02 + 1e-3).to(DEV)


def same_as_one_by_one(step, rounds=ROUNDS):
    """step(i, pause) runs round i, calls pause() between its kernels and returns what it made."""
    want = []
    for i in range(rounds):
        want.append([t.clone() for t in step(i, torch.cuda.synchronize)])
        torch.cuda.synchronize()
    got = [step(i, lambda: None) for i in range(rounds)]
    torch.cuda.synchronize()
    for i in range(rounds):
        for a, b in zip(got[i], want[i]):
            assert torch.equal(a, b), f"round {i}"


@pytest.mark.parametrize("cols", [33, 264, 1003])
@pytest.mark.parametrize("rows", [3, 64, 700])
def test_product_then_quantize(rows, cols):
    """Rows of C, off 16 bytes or on them, read by the quantization of the next kernel."""
    g = gen(rows + cols)
    K = 96
    a = [ints((rows, K), g) for _ in range(ROUNDS)]
    w, sa, sb = ints((cols, K), g).t(), scales((rows,), g), scales((cols,), g)
    c = torch.empty(rows, cols, dtype=torch.bfloat16, device=DEV)

    def step(i, pause):
        mb.scaled_mm(a[i], w, sa, sb, out=c)
        pause()
        return mb.quantize(c)
    same_as_one_by_one(step)


@pytest.mark.parametrize("cols", [40, 129, 1030])
def test_product_by_group_then_combine_and_gradients(cols):
    g = gen(cols)
    T, k, E, K = 50, 3, 6, 64
    o = mb.expert_sort(torch.randint(-1, E, (T, k), generator=g).to(DEV), E)
    a = [ints((T * k, K), g) for _ in range(ROUNDS)]
    w, sa, sb = ints((E, cols, K), g).transpose(1, 2), scales((T * k,), g), scales((E, cols), g)
    weights, d = torch.rand(T, k, generator=g).to(DEV), torch.randn(T, cols, generator=g).to(torch.bfloat16).to(DEV)
    y = torch.empty(T * k, cols, dtype=torch.bfloat16, device=DEV)

    def step(i, pause):
        mb.grouped_scaled_mm(a[i], w, sa, sb, o.offsets, out=y)
        pause()
        out = mb.expert_combine(y, weights, o)
        pause()
        return (out, *mb.expert_combine_backward(d, y, weights, o))
    same_as_one_by_one(step)


@pytest.mark.parametrize("rows,K,N", [(1, 2064, 300), (2, 500, 9000), (5, 1040, 600), (40, 500, 260)])
@pytest.mark.parametrize("start", [0, 1])
def test_quantize_then_product(rows, K, N, start):
    """Both operands fresh from the quantization, in storage that every round uses again; from
    column 1 on they are copied first."""
    g = gen(rows + K + N)
    x = [torch.randn(rows, K, generator=g).to(torch.bfloat16).to(DEV) for _ in range(ROUNDS)]
    w = [torch.randn(N, K, generator=g).to(torch.bfloat16).to(DEV) for _ in range(4)]

    def step(i, pause):
        q, s = mb.quantize(x[i])
        pause()
        wq, sw = mb.quantize(w[i % 4])
        pause()
        y = mb.scaled_mm(q[:, start:], wq[:, start:].t(), s, sw, out_dtype=torch.float32)
        pause()
        return (y,)
    same_as_one_by_one(step)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("K,N", [(640, 1024), (2048, 260)])
def test_products_with_one_row(dtype, K, N):
    """The row, the matrix (in both orientations) and the bias of a product, each made by the
    product before it."""
    g = gen(K + N)
    a = [torch.randn(1, 128, generator=g).to(dtype).to(DEV) for _ in range(ROUNDS)]
    b = torch.randn(128, K, generator=g).to(dtype).to(DEV)
    p = [torch.randn(K, 64, generator=g).to(dtype).to(DEV) for _ in range(4)]
    q = torch.randn(64, N, generator=g).to(dtype).to(DEV)
    x, w = torch.empty(1, K, dtype=dtype, device=DEV), torch.empty(K, N, dtype=dtype, device=DEV)
    wt = torch.empty(N, K, dtype=dtype, device=DEV)

    def step(i, pause):
        mb.matmul(a[i], b, out=x)
        pause()
        mb.matmul(p[i % 4], q, out=w)
        pause()
        y = mb.matmul(x, w)
        pause()
        mb.matmul(q.t(), p[i % 4].t(), out=wt)
        pause()
        z = mb.matmul(x, wt.t())
        pause()
        return y, z, mb.addmm(y[0], p[i % 4], q)
    same_as_one_by_one(step)
