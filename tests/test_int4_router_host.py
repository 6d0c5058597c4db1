"""CPU: the 4-bit products and the router.  The C structure matches its mirror, names are public,
what cannot be taken is refused before any launch, and the kernels load coherently."""
from __future__ import annotations

import ctypes
import os
import re
import subprocess

import pytest
import torch

import metalblas
import metalblas_b200 as mb
from metalblas_b200 import _lib, int4, router

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "metalblas_b200", "csrc")
NAMES = ("quantize_int4", "dequantize_int4", "int4_mm", "grouped_int4_mm", "expert_route", "expert_route_backward",
         "expert_balance", "expert_balance_backward", "ExpertBalance")

X, Q, S = torch.zeros(4, 64, dtype=torch.bfloat16), torch.zeros(8, 32, dtype=torch.uint8), torch.ones(8, 2)
OFF = torch.tensor([0, 4], dtype=torch.int32)
LOGITS, IDS = torch.zeros(4, 8), torch.zeros(4, 2, dtype=torch.int32)
BALANCE = mb.ExpertBalance(torch.zeros(()), torch.zeros(8, dtype=torch.int32), torch.zeros((), dtype=torch.int32))


def test_names_are_public_in_both_packages():
    for name in NAMES:
        assert getattr(mb, name) is getattr(metalblas, name)


def test_desc_layout_matches_c(tmp_path):
    fields = [f[0] for f in _lib.Int4Desc._fields_]
    body = "\n".join(f'printf("{f} %zu\\n", offsetof(mb_int4_desc, {f}));' for f in fields)
    prog = tmp_path / "off.c"
    prog.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "metalblas_b200.h"\n'
                    f'int main(void){{ {body} printf("sizeof %zu\\n", sizeof(mb_int4_desc)); return 0; }}\n')
    exe = tmp_path / "off"
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(prog), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split("\n")
    got = dict(line.split() for line in out if line)
    for f in fields:
        assert int(got[f]) == getattr(_lib.Int4Desc, f).offset, f
    assert int(got["sizeof"]) == ctypes.sizeof(_lib.Int4Desc)


@pytest.mark.parametrize("call", [
    lambda: mb.quantize_int4(X), lambda: mb.dequantize_int4(Q, S, 32), lambda: mb.int4_mm(X, Q, S, 32),
    lambda: mb.grouped_int4_mm(X, Q[None], S[None], OFF, 32), lambda: mb.expert_route(LOGITS, 2),
    lambda: mb.expert_route_backward(LOGITS[:, :2], LOGITS, IDS), lambda: mb.expert_balance(LOGITS, IDS),
    lambda: mb.expert_balance_backward(torch.ones(()), LOGITS, BALANCE)])
def test_cpu_tensors_are_refused(call):
    with pytest.raises(AssertionError):
        call()


@pytest.mark.parametrize("call", [
    lambda x: mb.quantize_int4(x), lambda x: mb.dequantize_int4(x, S, 32), lambda x: mb.int4_mm(x, Q, S, 32),
    lambda x: mb.grouped_int4_mm(x, Q[None], S[None], OFF, 32), lambda x: mb.expert_route(x, 2),
    lambda x: mb.expert_route_backward(x, x, IDS), lambda x: mb.expert_balance(x, IDS),
    lambda x: mb.expert_balance_backward(x, x, BALANCE),
    lambda x: int4._int4_mm.__wrapped__(X, x, S, 32, None, None, None, None),
    lambda x: int4._int4_mm.__wrapped__(X, Q, x, 32, None, None, None, None),
    lambda x: int4._int4_mm.__wrapped__(X, Q, S, 32, x, None, None, None),
    lambda x: int4._int4_mm.__wrapped__(X, Q, S, 32, None, x, None, None),
    lambda x: int4._int4_mm.__wrapped__(X, Q, S, 32, None, None, x, None),
    lambda x: int4._grouped_int4_mm.__wrapped__(X, Q[None], S[None], x, 32, None, None, None),
    lambda x: router._balance.__wrapped__(LOGITS, x, None), lambda x: router._balance.__wrapped__(LOGITS, IDS, x),
    lambda x: router._route_backward.__wrapped__(LOGITS, x, IDS, True)])
@pytest.mark.parametrize("x", [0.5, [1.0, 2.0], "x"])
def test_no_tensor(call, x):
    with pytest.raises(AssertionError):
        call(x)


def desc(**kw):
    d = _lib.Int4Desc()
    _lib.load().mb_int4_desc_init(ctypes.byref(d))
    d.dtype = d.scale_dtype = d.bias_dtype = _lib.MB_BF16
    d.group, d.M, d.N, d.K = 128, 8, 64, 256
    d.x = d.w = d.scale = d.out = 1 << 20   # aligned; nothing is launched on it
    d.x_rs, d.w_rs, d.scale_rs, d.out_rs, d.w_e, d.scale_e = 256, 128, 2, 64, 64 * 128, 128
    for name, v in kw.items():
        setattr(d, name, v)
    return d


@pytest.mark.parametrize("kw,code", [
    (dict(dtype=_lib.MB_F32), _lib.MB_ERR_UNSUPPORTED), (dict(scale_dtype=_lib.MB_F16), _lib.MB_ERR_UNSUPPORTED),
    (dict(group=48), _lib.MB_ERR_INVALID), (dict(M=-1), _lib.MB_ERR_INVALID), (dict(K=(1 << 30) + 1), _lib.MB_ERR_INVALID),
    (dict(groups=1025), _lib.MB_ERR_INVALID), (dict(groups=2), _lib.MB_ERR_INVALID), (dict(x=None), _lib.MB_ERR_INVALID),
    (dict(w=None), _lib.MB_ERR_INVALID), (dict(scale=None), _lib.MB_ERR_INVALID), (dict(out=None), _lib.MB_ERR_INVALID),
    (dict(out_rs=63), _lib.MB_ERR_INVALID), (dict(x_rs=255), _lib.MB_ERR_INVALID), (dict(w_rs=127), _lib.MB_ERR_INVALID),
    (dict(w_e=-1, groups=1, offsets=1 << 20), _lib.MB_ERR_INVALID),
    (dict(bias=1 << 20, bias_dtype=_lib.MB_F16), _lib.MB_ERR_INVALID)])
def test_c_entry_refuses(lib, kw, code):
    assert lib.mb_int4_gemm(ctypes.byref(desc(**kw)), None) == code
    assert _lib.last_error()
    assert lib.mb_int4_gemm(None, None) == _lib.MB_ERR_INVALID
    assert lib.mb_int4_workspace_size(ctypes.byref(desc(**kw))) == 0


def test_c_entries_of_rows_refuse(lib):
    p, F32, I32 = 1 << 20, _lib.MB_F32, _lib.MB_I32
    bad = _lib.MB_ERR_INVALID
    assert lib.mb_int4_quantize(I32, F32, 2, 64, 32, p, 64, p, 32, p, 2, None) == _lib.MB_ERR_UNSUPPORTED
    assert lib.mb_int4_quantize(F32, F32, 2, 64, 33, p, 64, p, 32, p, 2, None) == bad
    assert lib.mb_int4_quantize(F32, F32, 2, 64, 32, p, 63, p, 32, p, 2, None) == bad
    assert lib.mb_int4_quantize(F32, F32, 2, 64, 32, p, 64, p, 31, p, 2, None) == bad
    assert lib.mb_int4_quantize(F32, F32, 2, 64, 32, p, 64, p, 32, p, 1, None) == bad
    assert lib.mb_int4_quantize(F32, F32, 2, 64, 32, None, 64, p, 32, p, 2, None) == bad
    assert lib.mb_int4_quantize(F32, F32, 0, 64, 32, None, 64, None, 32, None, 2, None) == _lib.MB_OK
    assert lib.mb_int4_dequantize(F32, F32, 2, 64, 32, p, 32, p, 2, p, 1, p, 64, None) == bad
    assert lib.mb_expert_route(I32, 4, 8, 2, 1, p, 8, p, p, None) == _lib.MB_ERR_UNSUPPORTED
    assert lib.mb_expert_route(F32, 4, 8, 9, 1, p, 8, p, p, None) == bad
    assert lib.mb_expert_route(F32, 4, 1025, 2, 1, p, 1025, p, p, None) == bad
    assert lib.mb_expert_route(F32, 4, 8, 2, 1, p, 7, p, p, None) == bad
    assert lib.mb_expert_route(F32, 1 << 30, 8, 2, 1, p, 8, p, p, None) == bad
    assert lib.mb_expert_route_backward(F32, 4, 8, 2, 1, None, p, 8, p, p, None) == bad
    need = lib.mb_expert_balance_workspace_size(4, 8)
    assert need > 0
    assert lib.mb_expert_balance(F32, 4, 8, 2, p, 8, p, None, p, p, p, p, need - 1, None) == _lib.MB_ERR_WORKSPACE
    assert lib.mb_expert_balance(F32, 4, 8, 2, p, 8, p, None, p, p, p, p + 2, need, None) == _lib.MB_ERR_WORKSPACE
    assert lib.mb_expert_balance(F32, 4, 8, 2, p, 8, None, None, p, p, p, p, need, None) == bad
    assert lib.mb_expert_balance_backward(F32, 4, 8, None, p, 8, p, p, None, p, None) == bad


def test_plans_answer_without_a_device(lib):
    buf = ctypes.create_string_buffer(256)
    for kw in (dict(), dict(M=1), dict(M=4000, N=5000, out_rs=5000), dict(M=64, groups=8, offsets=1 << 20), dict(K=0), dict(M=0),
               dict(w_rs=129), dict(x_rs=257), dict(M=1, K=64)):
        assert lib.mb_int4_plan(ctypes.byref(desc(**kw)), buf, 256) > 0
        assert buf.value


@pytest.mark.parametrize("name", [f for f in sorted(os.listdir(CSRC)) if f.startswith(("int4", "router"))])
def test_kernels_load_coherently(name):
    """They may start beside their predecessor, and the wait for it orders ordinary loads alone."""
    with open(os.path.join(CSRC, name)) as f:
        code = re.sub(r"//[^\n]*", "", f.read())
    assert "ld.global.nc" not in code and "__ldg" not in code
