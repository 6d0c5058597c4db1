"""An ``out`` of the 4-bit products beside, and in the way of, what the call reads.

The inputs of tests/test_gpu_int4.py whose sums are exact: the result is the exact value rounded once."""
from __future__ import annotations

import pytest
import torch

import metalblas_b200 as mb
from tests.test_gpu_int4 import DEV, gen, split, tokens, unpacked, weights

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("M", [1, 3, 70])
@pytest.mark.parametrize("K,N", [(256, 96), (200, 77)])
def test_beside_the_tokens(M, K, N):
    """Tokens and results in one buffer, row beside row."""
    g = gen(M + K)
    q, s, _ = weights((N,), K, 64, g, torch.bfloat16, False, True)
    buf = torch.full((M, K + N + 3), 5.0, dtype=torch.bfloat16, device=DEV)
    x = buf[:, :K].copy_(tokens(M, K, g, torch.bfloat16, True))
    want = (x.double() @ unpacked(q, s, None, K, 64).t()).bfloat16()
    out = mb.int4_mm(x, q, s, 64, out=buf[:, K + 1:K + 1 + N])
    assert torch.equal(out, want) and bool((buf[:, K] == 5).all()) and bool((buf[:, K + 1 + N:] == 5).all())
    again = mb.grouped_int4_mm(x, q[None], s[None], split([M]), 64, out=buf[:, K + 2:K + 2 + N])
    assert torch.equal(again, want)


def test_in_the_way():
    K = 64
    q, s, z = weights((K,), K, 32, gen(0), torch.bfloat16, True, True)
    bias = torch.zeros(K, dtype=torch.bfloat16, device=DEV)
    for M in (1, 4, 90):
        x = tokens(M, K, gen(1), torch.bfloat16, True)
        before = x.clone()
        for call in (lambda: mb.int4_mm(x, q, s, 32, zero=z, out=x),
                     lambda: mb.grouped_int4_mm(x, q[None], s[None], split([M]), 32, out=x),
                     lambda: mb.int4_mm(x, q, s, 32, bias=bias, out=bias.view(1, K).expand(M, K)[:1]) if M == 1 else
                     mb.int4_mm(x, q, s, 32, out=x)):
            with pytest.raises(ValueError, match="share"):
                call()
        assert torch.equal(x, before) and not bool(bias.any())
