"""Products over an empty K by group: the rows' groups follow the same rules as with any K."""
from __future__ import annotations

import ctypes

import pytest
import torch

import metalblas_b200 as mb
from metalblas_b200 import _lib

pytestmark = pytest.mark.gpu
DEV = "cuda"
FLOATS = (torch.float32, torch.float16, torch.bfloat16)
M, N, E = 40, 24, 4
# (offsets, the group of each row or -1)
GOOD = [([0, 10, 10, 30, 40], [0] * 10 + [2] * 20 + [3] * 10), ([0, 0, 7, 7, 20], [1] * 7 + [3] * 13 + [-1] * 20),
        ([0, 0, 0, 0, 0], [-1] * M), ([0, 5, 9, 50, 60], [0] * 5 + [1] * 4 + [2] * 31)]
BAD = [[0, M, 0, M, 2], [0, 5, 3, M, M], [0, M, M, M, 0], [0, -5, 10, 9, M]]


def run(offsets, sa, sb, bias, out_dtype, K=0):
    """mb_scaled_gemm by group with a bias, through the descriptor."""
    lib = _lib.load()
    a = torch.ones(M, max(K, 16), dtype=torch.int8, device=DEV)[:, :K]
    b = torch.ones(E, N, max(K, 16), dtype=torch.int8, device=DEV)[:, :, :K]
    c = torch.full((M, N), 7.0, dtype=out_dtype, device=DEV)
    off = torch.tensor(offsets, dtype=torch.int32, device=DEV)
    d = _lib.ScaledDesc()
    lib.mb_scaled_desc_init(ctypes.byref(d))
    d.out_dtype = d.bias_dtype = _lib.DTYPE_CODE[out_dtype]
    d.M, d.N, d.K, d.groups = M, N, K, E
    d.A, d.B, d.C, d.offsets = a.data_ptr(), b.data_ptr(), c.data_ptr(), off.data_ptr()
    d.a_rs, d.a_cs, d.sB, d.b_rs, d.b_cs, d.c_rs, d.c_cs = a.stride(0), 1, b.stride(0), 1, b.stride(1), N, 1
    d.scale_a, d.scale_a_s, d.scale_b, d.scale_b_s, d.scale_b_g = sa.data_ptr(), 1, sb.data_ptr(), 1, N
    if bias is not None:
        d.bias, d.bias_s = bias.data_ptr(), 1
    _lib.raise_for(lib.mb_scaled_gemm(ctypes.byref(d), ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)))
    torch.cuda.synchronize()
    return c


def inputs(seed, dtype):
    g = torch.Generator().manual_seed(seed)
    return (torch.rand(M, generator=g).to(DEV) + 0.5, torch.rand(E, N, generator=g).to(DEV) + 0.5,
            torch.randn(N, generator=g).to(dtype).to(DEV))


@pytest.mark.parametrize("K", [0, 16])
@pytest.mark.parametrize("dtype", FLOATS)
def test_bias_by_group(dtype, K):
    """Exactly K + bias in the rows of groups (scales of one), zero in the others."""
    sa, sb, bias = torch.ones(M, device=DEV), torch.ones(E, N, device=DEV), inputs(1, dtype)[2]
    for offsets, group in GOOD:
        c = run(offsets, sa, sb, bias, dtype, K)
        live = torch.tensor([e >= 0 for e in group], device=DEV)[:, None]
        want = torch.where(live, (bias.float() + K).to(dtype).expand(M, N), torch.zeros((), dtype=dtype, device=DEV))
        assert torch.equal(c, want), offsets


@pytest.mark.parametrize("K", [0, 16])
@pytest.mark.parametrize("dtype", FLOATS)
def test_offsets_that_are_not_ascending(dtype, K):
    sa, sb, bias = inputs(2, dtype)
    sa[3] = float("nan")
    for offsets in BAD:
        assert bool((run(offsets, sa, sb, bias, dtype, K) == 0).all()), offsets


@pytest.mark.parametrize("K", [0, 16])
def test_scales_of_rows_without_a_group_are_not_used(K):
    """A scale that is no number shows in its own rows alone."""
    sa, sb, _ = inputs(3, torch.float32)
    sa[::3], sb[2, 5] = float("nan"), float("inf")
    for offsets, group in GOOD:
        c = run(offsets, sa, sb, None, torch.float32, K)
        for m, e in enumerate(group):
            if e < 0:
                assert bool((c[m] == 0).all())
            elif m % 3 == 0:
                assert bool(torch.isnan(c[m]).all())


def test_through_the_public_entry_point():
    sa, sb, _ = inputs(4, torch.float32)
    sa[:] = float("nan")
    a = torch.zeros(M, 0, dtype=torch.int8, device=DEV)
    b = torch.zeros(E, 0, N, dtype=torch.int8, device=DEV)
    for offsets, want_nan in ((GOOD[0][0], M), (GOOD[1][0], 20), (BAD[0], 0), (BAD[1], 0)):
        off = torch.tensor(offsets, dtype=torch.int32, device=DEV)
        y = mb.grouped_scaled_mm(a, b, sa, sb, off)
        assert int(torch.isnan(y).all(1).sum()) == want_nan
        assert bool((y[want_nan:] == 0).all())
