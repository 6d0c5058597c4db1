"""Where the int8 products may write: every layout of ``out`` that gives each element a place of
its own, and no other."""
from __future__ import annotations

import pytest
import torch

import metalblas_b200 as mb

pytestmark = pytest.mark.gpu
DEV = "cuda"
M, K, N, E = 12, 64, 40, 2


def make():
    g = torch.Generator().manual_seed(7)
    a = torch.randint(-127, 128, (M, K), dtype=torch.int8, generator=g).to(DEV)
    w = torch.randint(-127, 128, (E, N, K), dtype=torch.int8, generator=g).to(DEV).transpose(1, 2)
    sa, sb = torch.rand(M, generator=g).to(DEV), torch.rand(E, N, generator=g).to(DEV)
    return a, w, sa, sb, torch.tensor([0, 5, 12], dtype=torch.int32, device=DEV)


def test_outputs_that_share_memory_are_refused():
    a, w, sa, sb, off = make()
    room = torch.full((4 * M * N,), 7.0, device=DEV)
    for strides in ((0, 1), (1, 0), (0, 0), (N - 1, 1), (1, M - 1), (2, 4)):
        out = room.as_strided((M, N), strides)
        with pytest.raises(ValueError):
            mb.scaled_mm(a, w[0], sa, sb[0], out=out)
        with pytest.raises(ValueError):
            mb.grouped_scaled_mm(a, w, sa, sb, off, out=out)
    assert bool((room == 7).all())


def test_outputs_with_a_place_for_each_element():
    a, w, sa, sb, off = make()
    dense = mb.scaled_mm(a, w[0], sa, sb[0], out_dtype=torch.float32)
    grouped = mb.grouped_scaled_mm(a, w, sa, sb, off, out_dtype=torch.float32)
    for strides in ((N, 1), (1, M), (2 * N, 2), (2, 2 * M), (N + 3, 1), (3, 3 * M + 1), (N + 1, N * (N + 1) * M // N)):
        span = (M - 1) * strides[0] + (N - 1) * strides[1] + 1
        for call, want in ((lambda o: mb.scaled_mm(a, w[0], sa, sb[0], out=o), dense),
                           (lambda o: mb.grouped_scaled_mm(a, w, sa, sb, off, out=o), grouped)):
            room = torch.full((span + 8,), 7.0, device=DEV)
            out = room.as_strided((M, N), strides)
            assert torch.equal(call(out), want), strides
            out.fill_(7.0)
            assert bool((room == 7).all()), strides
    one = torch.full((1,), 7.0, device=DEV).expand(1, 1)  # a single element has any strides
    mb.scaled_mm(a[:1], w[0][:, :1], sa[:1], sb[0, :1], out=one)
    assert torch.equal(one, dense[:1, :1])


@pytest.mark.parametrize("plan", [None, (16, 1, 1, 1), (64, 2, 1, 1), (128, 1, 1, 1), (128, 1, -1, 1), (128, 4, -1, 1),
                                  (256, 1, -1, 1), (256, 1, -1, 2)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_transposed_outputs_by_group(dtype, plan):
    """Columns of C contiguous, with rows of no group at the end."""
    g = torch.Generator().manual_seed(9)
    K, E = 528, 5
    for counts, extra, N in (([3, 0, 70, 1, 20], 9, 300), ([0, 130, 5, 0, 200], 40, 261), ([2, 1, 0, 2, 1], 1, 515)):
        M = sum(counts) + extra
        a = torch.randint(-127, 128, (M, K), dtype=torch.int8, generator=g).to(DEV)
        w = torch.randint(-127, 128, (E, N, K), dtype=torch.int8, generator=g).to(DEV).transpose(1, 2)
        sa, sb = torch.rand(M, generator=g).to(DEV), torch.rand(E, N, generator=g).to(DEV)
        off = torch.tensor([0] + list(torch.tensor(counts).cumsum(0)), dtype=torch.int32, device=DEV)
        want = mb.grouped_scaled_mm(a, w, sa, sb, off, out_dtype=dtype)
        assert bool((want[M - extra:] == 0).all())
        for pitch in (M, M + 3):
            room = torch.full((N, pitch), 7.0, dtype=dtype, device=DEV)
            mb.grouped_scaled_mm(a, w, sa, sb, off, out=room[:, :M].t(), _plan=plan)
            assert torch.equal(room[:, :M].t(), want)
            assert bool((room[:, M:] == 7).all())
