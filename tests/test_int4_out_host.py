"""CPU: an ``out`` of the 4-bit products that shares memory with an operand is refused before any
launch: blocks would write results where others still read.  Rows beside one another in one buffer share
nothing; the rule is checked against sets of bytes."""
from __future__ import annotations

import ctypes
import random

import pytest

from metalblas_b200 import _lib
from tests.test_int4_router_host import desc

AT = 1 << 20


def refused(lib, d):
    """By the argument checks alone: the plan asks for a workspace (w off 16 bytes) that is not given,
    so nothing is launched either way."""
    code = lib.mb_int4_gemm(ctypes.byref(d), None)
    assert code in (_lib.MB_ERR_INVALID, _lib.MB_ERR_WORKSPACE), code
    return code == _lib.MB_ERR_INVALID


def apart(**kw):
    far = dict(w=(64 << 20) + 1, scale=128 << 20, out=192 << 20)
    return desc(**{**far, **kw})


def rows(at, count, pitch, size):
    return {b for m in range(count) for b in range(at + m * pitch, at + m * pitch + size)}


def test_tokens(lib):
    rng = random.Random(5)
    seen = set()
    for _ in range(4000):
        M, K, N = rng.randint(1, 5), rng.randint(1, 12), rng.randint(1, 12)
        xr, pitch = K + rng.choice((0, 1, 5, 16)), N + rng.choice((0, 1, 5, 16))
        if rng.random() < 0.5:
            pitch = max(xr, N)
            xr = max(pitch, K)
            pitch = xr
        at = 2 * rng.randint(-60, 60)
        both = rows(AT, M, 2 * xr, 2 * K) & rows(AT + at, M, 2 * pitch, 2 * N)
        d = apart(M=M, K=K, N=N, x=AT, x_rs=xr, out=AT + at, out_rs=pitch, w_rs=(K + 1) // 2 + 1, scale_rs=1)
        assert refused(lib, d) == bool(both), (M, K, N, xr, pitch, at)
        seen.add(bool(both))
    assert seen == {True, False}


@pytest.mark.parametrize("kw,bad", [
    (dict(), False), (dict(bias=AT), False), (dict(bias=(192 << 20) + 2), True), (dict(bias=(192 << 20) - 2 * 64), False),
    (dict(bias=(192 << 20) - 2), True), (dict(scale=192 << 20), True), (dict(scale=(192 << 20) - 4), True),
    (dict(w=(192 << 20) + 1), True), (dict(zero=192 << 20, zero_rs=2), True), (dict(zero=AT * 3, zero_rs=2), False),
    (dict(out_rs=128, bias=(192 << 20) + 128), False)])
def test_other_operands(lib, kw, bad):
    d = apart(x=AT, **kw)
    assert refused(lib, d) == bad
    if bad:
        assert "share" in _lib.last_error()


def test_matrices_by_group(lib):
    one = dict(x=AT, groups=3, offsets=AT * 2, w=(64 << 20) + 1, w_rs=129, w_e=64 * 129)
    assert not refused(lib, apart(**one))
    assert refused(lib, apart(**one, out=(64 << 20) + 2 * 64 * 129 + 5))       # in the last matrix
    assert not refused(lib, apart(**one, out=(64 << 20) + 2 + 3 * 64 * 129))
    assert refused(lib, apart(**one, out=AT * 2 + 12)) and not refused(lib, apart(**one, out=AT * 2 + 16))
