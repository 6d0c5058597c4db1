"""CPU: the C structure of the int8 products matches its mirror, the entry points refuse what
they cannot take before any launch, and the plans answer without a device."""
from __future__ import annotations

import ctypes
import os
import subprocess

import pytest
import torch

import metalblas
import metalblas_b200 as mb
from metalblas_b200 import _lib

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
NAMES = ("quantize", "scaled_mm", "grouped_scaled_mm", "ExpertOrder", "expert_sort", "expert_gather",
         "expert_gather_quantize", "expert_combine", "expert_gather_backward", "expert_combine_backward")


def test_names_are_public_in_both_packages():
    for name in NAMES:
        assert getattr(mb, name) is getattr(metalblas, name)


def test_scaled_desc_layout_matches_c(tmp_path):
    fields = [f[0] for f in _lib.ScaledDesc._fields_]
    body = "\n".join(f'printf("{f} %zu\\n", offsetof(mb_scaled_desc, {f}));' for f in fields)
    prog = tmp_path / "off.c"
    prog.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "metalblas_b200.h"\n'
                    f'int main(void){{ {body} printf("sizeof %zu\\n", sizeof(mb_scaled_desc)); return 0; }}\n')
    exe = tmp_path / "off"
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(prog), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split("\n")
    got = dict(line.split() for line in out if line)
    for f in fields:
        assert int(got[f]) == getattr(_lib.ScaledDesc, f).offset, f
    assert int(got["sizeof"]) == ctypes.sizeof(_lib.ScaledDesc)


def test_cpu_tensors_are_refused():
    i8, f = torch.zeros(4, 16, dtype=torch.int8), torch.ones(4)
    ids = torch.zeros(4, 2, dtype=torch.int64)
    order = mb.ExpertOrder(torch.zeros(8, dtype=torch.int32), torch.zeros(4, 2, dtype=torch.int32),
                           torch.zeros(3, dtype=torch.int32))
    for call in (lambda: mb.quantize(torch.zeros(2, 2)), lambda: mb.scaled_mm(i8, i8.t(), f, f),
                 lambda: mb.grouped_scaled_mm(i8, i8.t()[None], f, f[None], order.offsets[:2]),
                 lambda: mb.expert_sort(ids, 4), lambda: mb.expert_gather(torch.zeros(4, 8), order),
                 lambda: mb.expert_gather_quantize(torch.zeros(4, 8), order),
                 lambda: mb.expert_combine(torch.zeros(8, 8), None, order),
                 lambda: mb.expert_gather_backward(torch.zeros(8, 8), order),
                 lambda: mb.expert_combine_backward(torch.zeros(4, 8), torch.zeros(8, 8), torch.ones(4, 2), order)):
        with pytest.raises(AssertionError):
            call()


def desc(M=64, K=256, N=128, groups=0, **kw):
    d = _lib.ScaledDesc()
    _lib.load().mb_scaled_desc_init(ctypes.byref(d))
    d.out_dtype = d.bias_dtype = _lib.MB_BF16
    d.M, d.N, d.K, d.groups = M, N, K, groups
    d.A = d.B = d.C = d.scale_a = d.scale_b = 1 << 20   # aligned; nothing is launched on it
    d.a_rs, d.a_cs, d.b_rs, d.b_cs, d.sB, d.c_rs, d.c_cs = K, 1, 1, K, N * K, N, 1
    d.scale_a_s = d.scale_b_s = 1
    d.scale_b_g = N
    if groups:
        d.offsets = 1 << 20
    for name, v in kw.items():
        setattr(d, name, v)
    return d


@pytest.mark.parametrize("kw,code", [
    (dict(out_dtype=_lib.MB_I8), _lib.MB_ERR_UNSUPPORTED), (dict(K=131072), _lib.MB_ERR_INVALID),
    (dict(M=-1), _lib.MB_ERR_INVALID), (dict(groups=1025), _lib.MB_ERR_INVALID),
    (dict(groups=2, offsets=None), _lib.MB_ERR_INVALID), (dict(C=None), _lib.MB_ERR_INVALID),
    (dict(A=None), _lib.MB_ERR_INVALID), (dict(scale_b=None), _lib.MB_ERR_INVALID),
    (dict(bias=1 << 20, bias_s=1, bias_dtype=_lib.MB_F16), _lib.MB_ERR_INVALID)])
def test_c_entry_refuses(lib, kw, code):
    assert lib.mb_scaled_gemm(ctypes.byref(desc(**kw)), None) == code
    assert _lib.last_error()
    assert lib.mb_scaled_gemm(None, None) == _lib.MB_ERR_INVALID


def test_c_entries_of_the_rows_refuse(lib):
    p = 1 << 20
    assert lib.mb_quantize(_lib.MB_I32, 2, 2, p, 2, p, 2, p, None) == _lib.MB_ERR_UNSUPPORTED
    assert lib.mb_quantize(_lib.MB_F32, -1, 2, p, 2, p, 2, p, None) == _lib.MB_ERR_INVALID
    assert lib.mb_quantize(_lib.MB_F32, 2, 4, p, 3, p, 4, p, None) == _lib.MB_ERR_INVALID
    assert lib.mb_quantize(_lib.MB_F32, 2, 4, None, 4, p, 4, p, None) == _lib.MB_ERR_INVALID
    assert lib.mb_quantize(_lib.MB_F32, 0, 4, None, 4, None, 4, None, None) == _lib.MB_OK
    assert lib.mb_expert_sort(0, 4, 0, p, p, p, p, None) == _lib.MB_ERR_INVALID
    assert lib.mb_expert_sort(0, 4, 1025, p, p, p, p, None) == _lib.MB_ERR_INVALID
    assert lib.mb_expert_sort(0, 1 << 31, 4, p, p, p, p, None) == _lib.MB_ERR_INVALID
    assert lib.mb_expert_gather(_lib.MB_F32, 1 << 30, 4, 4, p, 4, p, p, p, 4, None) == _lib.MB_ERR_INVALID
    assert lib.mb_expert_gather(_lib.MB_F32, 4, 2, 4, p, 4, None, p, p, 4, None) == _lib.MB_ERR_INVALID
    assert lib.mb_expert_combine(_lib.MB_F32, _lib.MB_F16, 4, 2, 4, p, 4, p, p, p, p, 4, None) == \
        _lib.MB_ERR_UNSUPPORTED
    assert lib.mb_expert_combine_backward(_lib.MB_F16, _lib.MB_F32, 4, 2, 4, p, 4, p, 4, None, p, p, p, 4, p, None) == \
        _lib.MB_ERR_INVALID


def test_plans_answer_without_a_device(lib):
    buf = ctypes.create_string_buffer(256)
    for kw in (dict(), dict(M=1), dict(M=5000, N=5000, K=4096), dict(M=64, groups=8), dict(M=9000, groups=3), dict(K=0),
               dict(M=0), dict(a_rs=257), dict(b_cs=257)):
        assert lib.mb_scaled_plan(ctypes.byref(desc(**kw)), buf, 256) > 0
        assert buf.value
