"""Scratch of a C caller: on the boundary the plan's kernels need, or refused before a launch."""
from __future__ import annotations

import ctypes

import pytest
import torch

import metalblas_b200 as mb
from metalblas_b200 import _lib, kernels

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(autouse=True)
def no_wait_gave_up():
    yield
    torch.cuda.synchronize()
    assert kernels.device_status() == 0


def product(lib, a, b, c):
    d = _lib.new_desc()
    d.dtype = _lib.DTYPE_CODE[a.dtype]
    (d.M, d.K), d.N = a.shape, b.shape[1]
    d.A, d.B, d.C = a.data_ptr(), b.data_ptr(), c.data_ptr()
    (d.a_rs, d.a_cs), (d.b_rs, d.b_cs), (d.c_rs, d.c_cs) = a.stride(), b.stride(), c.stride()
    d.workspace_bytes = -1
    need = int(lib.mb_gemm_workspace_size(ctypes.byref(d)))
    d.workspace_bytes = need
    return d, need


CASES = [("split-K", torch.bfloat16, 16, 4096, 1024, 0), ("copied operand", torch.bfloat16, 1024, 1024, 1024, 1),
         ("3xTF32", torch.float32, 256, 512, 256, 0), ("byte planes", torch.int32, 512, 512, 512, 0)]


@pytest.mark.parametrize("name,dtype,M,K,N,start", CASES, ids=[c[0] for c in CASES])
def test_scratch_of_products(lib, name, dtype, M, K, N, start):
    g = torch.Generator().manual_seed(M + K)
    make = lambda *s: (torch.randint(-9, 9, s, generator=g) if dtype is torch.int32  # noqa: E731
                       else torch.randn(s, generator=g)).to(dtype).to(DEV)
    a, b, c = make(M, K + start)[:, start:], make(K, N), torch.zeros(M, N, dtype=dtype, device=DEV)
    d, need = product(lib, a, b, c)
    if name == "split-K":
        d.backend, d.split_k, d.cta_pair, d.swap_ab, d.tile_n = _lib.MB_BACKEND_TC, 3, 1, -1, 128
        d.workspace_bytes = -1
        need = d.workspace_bytes = int(lib.mb_gemm_workspace_size(ctypes.byref(d)))
    assert need > 0
    ws = torch.zeros(need + 64, dtype=torch.uint8, device=DEV)
    stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    for off in (1, 2, 4, 8, 12):
        d.workspace = ws.data_ptr() + off
        assert lib.mb_gemm(ctypes.byref(d), stream) == _lib.MB_ERR_WORKSPACE
        assert "16-byte" in _lib.last_error()
    torch.cuda.synchronize()
    assert not bool(c.any()) and not bool(ws.any())
    d.workspace = ws.data_ptr() + 16
    _lib.raise_for(lib.mb_gemm(ctypes.byref(d), stream))
    want, size = a.double() @ b.double(), a.double().abs() @ b.double().abs()
    if dtype is torch.int32:
        assert torch.equal(c.double(), want)
    else:  # K fp32 roundings, and one of the type (3xTF32: 2^-20 a product)
        unit = 2.0 ** -8 if dtype is torch.bfloat16 else 2.0 ** -20
        assert bool(((c.double() - want).abs() <= size * (K * 2.0 ** -24 + unit)).all())


def test_scratch_of_scaled_products(lib):
    """mb_scaled_gemm the same; scratch that nothing uses may lie anywhere."""
    g = torch.Generator().manual_seed(1)
    M, K, N = 64, 256, 128
    A = torch.randint(-127, 128, (M, K + 16), dtype=torch.int8, generator=g).to(DEV)
    b = torch.randint(-127, 128, (N, K), dtype=torch.int8, generator=g).to(DEV).t()
    sa, sb = torch.rand(M, generator=g).to(DEV), torch.rand(N, generator=g).to(DEV)
    stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    for start in (0, 1):
        a, c = A[:, start:start + K], torch.zeros(M, N, device=DEV)
        d = _lib.ScaledDesc()
        d.out_dtype = d.bias_dtype = _lib.MB_F32
        d.M, d.N, d.K = M, N, K
        d.A, d.B, d.C = a.data_ptr(), b.data_ptr(), c.data_ptr()
        (d.a_rs, d.a_cs), (d.b_rs, d.b_cs), (d.c_rs, d.c_cs) = a.stride(), b.stride(), c.stride()
        d.scale_a, d.scale_b, d.scale_a_s, d.scale_b_s = sa.data_ptr(), sb.data_ptr(), 1, 1
        need = int(lib.mb_scaled_workspace_size(ctypes.byref(d)))
        assert (need > 0) == (start == 1)
        ws = torch.zeros(need + 64, dtype=torch.uint8, device=DEV)
        d.workspace, d.workspace_bytes = ws.data_ptr() + 8, need
        rc = lib.mb_scaled_gemm(ctypes.byref(d), stream)
        if start:
            assert rc == _lib.MB_ERR_WORKSPACE
            torch.cuda.synchronize()
            assert not bool(c.any()) and not bool(ws.any())
            d.workspace = ws.data_ptr() + 16
            rc = lib.mb_scaled_gemm(ctypes.byref(d), stream)
        _lib.raise_for(rc, "mb_scaled_gemm")
        assert torch.equal(c, mb.scaled_mm(a.contiguous(), b, sa, sb, out_dtype=torch.float32))
