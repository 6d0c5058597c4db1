"""Operand layouts of the int8 products beside rows and columns of one matrix, and calls from two
threads at once."""
from __future__ import annotations

import threading

import pytest
import torch

import metalblas_b200 as mb
from metalblas_b200 import kernels

pytestmark = pytest.mark.gpu
DEV = "cuda"


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


@pytest.mark.parametrize("M", [1, 2, 9, 40, 300])
def test_rows_that_overlap(M):
    """Windows over one run of bytes: a row every 16, 48 or 5 bytes."""
    g = gen(M)
    K, N = 256, 96
    run, w, sa, sb = ints((16 * 400 + K,), g), ints((N, K), g).t(), scales((M,), g), scales((N,), g)
    for step in (16, 5, 0):
        a = run.as_strided((M, K), (step, 1))
        assert torch.equal(mb.scaled_mm(a, w, sa, sb), mb.scaled_mm(a.contiguous(), w, sa, sb))
    for step in (16, 5, 0):
        b = run.as_strided((N, K), (step, 1)).t()
        a = ints((M, K), g)
        assert torch.equal(mb.scaled_mm(a, b, sa, sb), mb.scaled_mm(a, b.t().contiguous().t(), sa, sb))


@pytest.mark.parametrize("counts", [[1, 0, 2], [5, 30, 0], [150, 3, 140]])
def test_weights_of_experts_side_by_side(counts):
    """Expert e's rows every E rows, or its columns every E columns."""
    g = gen(sum(counts))
    E, K, N, M = 3, 160, 112, sum(counts)
    a, sa, sb = ints((M, K), g), scales((M,), g), scales((E, N), g)
    off = torch.tensor([0] + list(torch.tensor(counts).cumsum(0)), dtype=torch.int32, device=DEV)
    W = ints((E, N, K), g)
    want = mb.grouped_scaled_mm(a, W.transpose(1, 2), sa, sb, off)
    by_row = W.transpose(0, 1).contiguous()                        # [N, E, K]
    assert torch.equal(mb.grouped_scaled_mm(a, by_row.permute(1, 2, 0), sa, sb, off), want)
    by_column = W.permute(1, 2, 0).contiguous()                    # [N, K, E]
    assert torch.equal(mb.grouped_scaled_mm(a, by_column.permute(2, 1, 0), sa, sb, off), want)
    by_k = W.permute(2, 0, 1).contiguous()                         # [K, E, N]
    assert torch.equal(mb.grouped_scaled_mm(a, by_k.permute(1, 0, 2), sa, sb, off), want)
    flipped = W.flip(0).contiguous()
    assert torch.equal(mb.grouped_scaled_mm(a, flipped.flip(0).transpose(1, 2), sa, sb, off), want)


def test_two_threads():
    """Each on a stream of its own, with shapes that set kernels up for the first time."""
    def work(seed, out):
        g = gen(seed)
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            for i in range(20):
                T, k, E, K, N = 30 + 17 * i, 2, 8, 64 + 16 * seed, 200
                ids = torch.randint(-1, E, (T, k), generator=g).to(DEV)
                x = torch.randn(T, K, generator=g).to(torch.bfloat16).to(DEV)
                w, sw = mb.quantize(torch.randn(E, N, K, generator=g).to(DEV))
                o = mb.expert_sort(ids, E)
                q, s = mb.expert_gather_quantize(x, o)
                y = mb.grouped_scaled_mm(q, w.transpose(1, 2), s, sw, o.offsets)
                out.append(mb.expert_combine(y, torch.rand(T, k, generator=g).to(DEV), o))
        stream.synchronize()

    want, got = {}, {1: [], 2: []}
    for seed in (1, 2):
        want[seed] = []
        work(seed, want[seed])
    threads = [threading.Thread(target=work, args=(seed, got[seed])) for seed in (1, 2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for seed in (1, 2):
        assert len(got[seed]) == 20 and all(torch.equal(x, y) for x, y in zip(got[seed], want[seed]))
