"""The one-pass kernel where the scales of a block's rows do not fit at once: it goes over the weights'
columns in several passes, each with scales and a ring of its own, and sums carry over.

Exact inputs (tests/test_gpu_int4.py): tokens up to 3, |u - zero| up to 15, scales 1/4 to 2, so a sum over K
columns is a multiple of 1/4 below K x 90, exact in fp32 for K up to 46000; every plan gives the same bits."""
from __future__ import annotations

import pytest
import torch

import metalblas_b200 as mb
from metalblas_b200 import kernels
from tests.test_gpu_int4 import DEV, TOKENS, gen, split, tokens, unpacked, weights

pytestmark = pytest.mark.gpu
WORDS = 15360        # fp32 words of scales that a block keeps


def passes(rows, K, G, zero):
    """Passes over the columns of a block that has `rows` weight rows of one unit."""
    tiles, per = min(7, -(-rows // 16)), max(1, 256 // G)
    fit = max(1, (WORDS // (2 if zero else 1) // (tiles * 16) - 1) // per)
    return -(-(-(-K // 256)) // fit)


@pytest.mark.parametrize("K,G,zero,least", [(17413, 32, False, 5), (17413, 32, True, 9), (17413, 64, True, 5),
                                            (17413, 128, True, 3), (18000, 128, False, 2), (35100, 256, True, 2), (2100, 32, True, 2)])
@pytest.mark.parametrize("M", [1, 11])
@pytest.mark.parametrize("dtype", TOKENS)
def test_dense(K, G, zero, least, M, dtype):
    N = 14336            # 97 rows a block: seven row tiles
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    assert sms != 148 or passes(-(-N // sms), K, G, zero) >= least
    g = gen(K + G)
    q, s, z = weights((N,), K, G, g, dtype, zero, True)
    x = tokens(M, K, g, dtype, True)
    want = torch.cat([x.double() @ unpacked(q[n:n + 2048], s[n:n + 2048], None if z is None else z[n:n + 2048], K, G).t()
                      for n in range(0, N, 2048)], 1).to(dtype)
    for plan in (None, (1, 0, 0, 0), (2, 0, 0, 0)):
        for _ in range(3):
            got = mb.int4_mm(x, q, s, G, zero=z, _plan=plan)
            assert torch.equal(got, want), (plan, int((got != want).sum()))
    assert kernels.device_status() == 0


@pytest.mark.parametrize("K,G,zero", [(8453, 32, True), (17413, 32, False), (17413, 128, True)])
@pytest.mark.parametrize("counts", [[1, 0, 9, 3], [20, 5, 0, 17]])
def test_by_group(K, G, zero, counts):
    """Units of several matrices, whose ends fall inside blocks: from seven row tiles to one."""
    N, dtype = 4001, torch.bfloat16
    g = gen(K + sum(counts))
    E, M = len(counts), sum(counts) + 2
    q, s, z = weights((E, N), K, G, g, torch.float32, zero, True)
    x = tokens(M, K, g, dtype, True)
    off = split(counts)
    want = torch.zeros(M, N, dtype=torch.float64, device=DEV)
    at = 0
    for e, c in enumerate(counts):
        want[at:at + c] = x[at:at + c].double() @ unpacked(q[e], s[e], None if z is None else z[e], K, G).t()
        at += c
    for plan in (None, (1, 0, 0, 0), (2, 0, 0, 0)):
        for _ in range(3):
            got = mb.grouped_int4_mm(x, q, s, off, G, zero=z, _plan=plan)
            assert torch.equal(got, want.to(dtype)), (plan, int((got != want.to(dtype)).sum()))
    assert kernels.device_status() == 0
