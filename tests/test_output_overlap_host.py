"""CPU: an output whose elements share memory is refused before any launch (its rows or columns
would race for one place), and every layout without such a pair passes that check."""
from __future__ import annotations

import ctypes
import itertools

import pytest

from metalblas_b200 import _lib
from tests.test_ops_host import desc


def overlaps(M, N, rs, cs):
    seen = [i * rs + j * cs for i, j in itertools.product(range(M), range(N))]
    return len(set(seen)) < len(seen)


STRIDES = (-40, -9, -4, -1, 0, 1, 2, 3, 4, 6, 7, 8, 9, 12, 40)


@pytest.mark.parametrize("M,N", [(1, 1), (1, 5), (5, 1), (2, 2), (3, 8), (8, 3), (5, 7)])
def test_c_with_elements_in_one_place(lib, M, N):
    """mb_scaled_plan runs the argument checks of mb_scaled_gemm and launches nothing."""
    buf = ctypes.create_string_buffer(256)
    for rs, cs in itertools.product(STRIDES, STRIDES):
        rc = lib.mb_scaled_plan(ctypes.byref(desc(M=M, N=N, c_rs=rs, c_cs=cs)), buf, 256)
        if overlaps(M, N, rs, cs):
            assert rc == -_lib.MB_ERR_INVALID, (rs, cs)
            assert lib.mb_scaled_gemm(ctypes.byref(desc(M=M, N=N, c_rs=rs, c_cs=cs)), None) == _lib.MB_ERR_INVALID
            assert "share" in _lib.last_error()
        else:
            assert rc > 0, (rs, cs)


def test_no_element_no_overlap(lib):
    buf = ctypes.create_string_buffer(256)
    for M, N in ((0, 5), (5, 0)):
        assert lib.mb_scaled_plan(ctypes.byref(desc(M=M, N=N, c_rs=0, c_cs=0)), buf, 256) > 0
