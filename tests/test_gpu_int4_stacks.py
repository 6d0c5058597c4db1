"""4-bit weights by group in stacks of other orders and of the smallest sizes: matrices row beside row
(the stride from matrix to matrix is smaller than from row to row), every other matrix, matrices of one row,
one matrix for all; and weights written anew between products, and products on two streams at once."""
from __future__ import annotations

import pytest
import torch

import metalblas_b200 as mb
from metalblas_b200 import kernels
from tests.test_gpu_int4 import DEV, gen, split, tokens, unpacked, weights

pytestmark = pytest.mark.gpu


def product(x, q, s, z, counts, K, G):
    want = torch.zeros(x.shape[0], q.shape[1], dtype=torch.float64, device=DEV)
    at = 0
    for e, c in enumerate(counts):
        want[at:at + c] = x[at:at + c].double() @ unpacked(q[e], s[e], None if z is None else z[e], K, G).t()
        at += c
    return want.to(x.dtype)


@pytest.mark.parametrize("counts", [[2, 0, 3, 1], [40, 3, 0, 90]])
@pytest.mark.parametrize("K,N,G", [(512, 200, 128), (96, 1, 32), (2048, 1, 64), (90, 2, 32), (1000, 33, 256)])
@pytest.mark.parametrize("zero", [False, True])
def test_orders(counts, K, N, G, zero):
    g = gen(K + N + sum(counts))
    E, M = len(counts), sum(counts) + 1
    q, s, z = weights((E, N), K, G, g, torch.bfloat16, zero, True)
    x = tokens(M, K, g, torch.bfloat16, True)
    off = split(counts)
    want = product(x, q, s, z, counts, K, G)

    def pitched(t):          # [N, E, pitch] underneath
        wide = torch.empty((N, E, (t.shape[2] + 15) // 16 * 16), dtype=t.dtype, device=DEV)
        return wide[..., :t.shape[2]].copy_(t.transpose(0, 1)).transpose(0, 1)

    def spread(t):           # every other matrix
        wide = torch.full((2 * E, t.shape[1], t.shape[2]), 3, dtype=t.dtype, device=DEV)
        wide[::2] = t
        return wide[::2]

    for change in (lambda t: t, pitched, spread, lambda t: t.contiguous(), lambda t: t.transpose(1, 2).contiguous().transpose(1, 2)):
        a = (change(q), change(s), None if z is None else change(z))
        for plan in (None, (1, 0, 0, 0), (2, 0, 0, 0), (16, 1, 0, 0), (128, 1, 0, 0), (256, 1, 0, 0)):
            got = mb.grouped_int4_mm(x, a[0], a[1], off, G, zero=a[2], _plan=plan)
            assert torch.equal(got, want), plan
    one = [t if t is None else t[:1].expand(E, *t.shape[1:]) for t in (q, s, z)]
    assert torch.equal(mb.grouped_int4_mm(x, one[0], one[1], off, G, zero=one[2]), product(x, one[0], one[1], one[2], counts, K, G))
    # one weight matrix, each group its own scales
    same = [one[0], s, z]
    assert torch.equal(mb.grouped_int4_mm(x, same[0], same[1], off, G, zero=same[2]), product(x, same[0], s, z, counts, K, G))
    assert kernels.device_status() == 0


def test_written_and_read_at_once():
    """Weights made, multiplied and made anew in a row, without a pause: each product has those before it."""
    g = torch.Generator(device=DEV).manual_seed(3)
    N, K, G = 3000, 2048, 128
    mats = [torch.randn(N, K, generator=g, device=DEV).bfloat16() for _ in range(3)]
    for M in (1, 12, 200):
        x = torch.randn(M, K, generator=g, device=DEV).bfloat16()
        want = []
        for w in mats:
            torch.cuda.synchronize()
            q, s = mb.quantize_int4(w, G)
            torch.cuda.synchronize()
            want.append(mb.int4_mm(x, q, s, G))
        q, s = (t.clone() for t in mb.quantize_int4(mats[0], G))
        torch.cuda.synchronize()
        for _ in range(20):
            got = []
            for w in mats:
                a, b = mb.quantize_int4(w, G)
                q.copy_(a)
                s.copy_(b)
                got.append(mb.int4_mm(x, q, s, G))
                got.append(mb.int4_mm(x, a, b, G))
            assert all(torch.equal(v, want[i // 2]) for i, v in enumerate(got))
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    outs = [[], []]
    for _ in range(20):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                outs[i].append(mb.int4_mm(x, q, s, G))
    torch.cuda.synchronize()
    assert all(torch.equal(v, want[2]) for o in outs for v in o)
    assert kernels.device_status() == 0
