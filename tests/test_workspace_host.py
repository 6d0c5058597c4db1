"""CPU: scratch that does not start on a 16-byte boundary is refused before any launch (the
kernels that fill it store sixteen bytes at a time)."""
from __future__ import annotations

import ctypes

import pytest

from metalblas_b200 import _lib
from tests.test_ops_host import desc

BASE = 1 << 20   # an aligned address; nothing is launched on it


@pytest.mark.parametrize("kw", [dict(a_rs=257), dict(b_cs=257), dict(a_cs=2, a_rs=512), dict(b_rs=2, b_cs=512),
                                dict(a_rs=257, b_cs=257, groups=4, sB=128 * 257)])
@pytest.mark.parametrize("off", [1, 2, 4, 8, 15])
def test_unaligned_scratch_is_refused(lib, kw, off):
    d = desc(**kw)
    need = lib.mb_scaled_workspace_size(ctypes.byref(d))
    assert need > 0
    d.workspace, d.workspace_bytes = BASE + off, need
    assert lib.mb_scaled_gemm(ctypes.byref(d), None) == _lib.MB_ERR_WORKSPACE
    assert "16-byte" in _lib.last_error()
