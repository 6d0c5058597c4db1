"""CPU: the line on a plan of the 4-bit products names every copy that the call makes first."""
from __future__ import annotations

import ctypes

import pytest

from tests.test_int4_router_host import desc


@pytest.mark.parametrize("M", [1, 8, 4000])
@pytest.mark.parametrize("plan", [(1, 0), (16, 1)])
@pytest.mark.parametrize("kw,copied", [(dict(), ()), (dict(x_rs=257), ("pack_x",)), (dict(w_rs=129), ("pack_w",)),
                                       (dict(x=(1 << 20) + 2), ("pack_x",)), (dict(x_rs=257, w_rs=129), ("pack_x", "pack_w"))])
def test_copies_are_named(lib, M, plan, kw, copied):
    d = desc(M=M, **kw)
    d.plan[:2] = plan
    if M == 1 and "x" not in kw:
        copied = tuple(c for c in copied if c != "pack_x")   # one row has no stride
    buf = ctypes.create_string_buffer(256)
    assert lib.mb_int4_plan(ctypes.byref(d), buf, 256) > 0
    line = buf.value.decode()
    for name in ("pack_x", "pack_w"):
        assert f"{name}={int(name in copied)}" in line, line
    assert (lib.mb_int4_workspace_size(ctypes.byref(d)) > 0) == bool(copied)
