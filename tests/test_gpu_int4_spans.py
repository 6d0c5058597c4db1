"""Conversions to 4 bits and back at the sizes of weight matrices, where a warp takes four spans of 256
columns at a time, and at one span beside them: every element against the definition in 64 bits.

Nothing is bounded here: scales, integers and values are equal.  A scale is amax / 7 in fp32 and then in
its type, a quotient of two numbers of at most 24 bits is a half or farther from one than a 64-bit
division is off, and a weight read back is a product in fp32 (exact in 64 bits) and then in its type.
"""
from __future__ import annotations

import math

import pytest
import torch

import metalblas_b200 as mb

pytestmark = pytest.mark.gpu
DEV = "cuda"
FLOATS = (torch.float32, torch.float16, torch.bfloat16)
NAN, INF = math.nan, math.inf


def definition(w, G, scale_dtype):
    """(integers u - 8 in 64 bits [rows, cols], scales)."""
    rows, K = w.shape
    groups = (K + G - 1) // G
    parts = torch.zeros(rows, groups * G, dtype=torch.float64, device=DEV)
    parts[:, :K] = w.double()
    parts = parts.view(rows, groups, G)
    amax = parts.abs().amax(2)                       # (NaN where a group holds one)
    scale = torch.where(amax.isfinite(), (amax / 7).float().to(scale_dtype), torch.tensor(NAN, dtype=scale_dtype, device=DEV))
    step = scale.double()[..., None]
    usable = step.isfinite() & (step > 0)
    q = torch.where(usable, torch.round(parts / torch.where(usable, step, 1.0)), 0.0).clamp(-7, 7)
    return q.view(rows, -1)[:, :K], scale


def integers(q, K):
    return torch.stack((q & 15, q >> 4), -1).reshape(q.shape[0], -1)[:, :K].double() - 8


def check(w, G, scale_dtype, outs=FLOATS):
    q, s = mb.quantize_int4(w, G, scale_dtype=scale_dtype)
    want, scale = definition(w, G, scale_dtype)
    assert torch.equal(torch.nan_to_num(s.double(), nan=-1.0), torch.nan_to_num(scale.double(), nan=-1.0))
    K = w.shape[1]
    got = integers(q, K)
    assert torch.equal(got, want), f"{int((got != want).sum())} of {got.numel()} differ"
    values = want * scale.double().repeat_interleave(G, 1)[:, :K]
    for out in outs:
        back = mb.dequantize_int4(q, s, G, cols=K, out_dtype=out)
        assert torch.allclose(back, values.float().to(out), rtol=0, atol=0, equal_nan=True)
    return q, s


# Four spans a task from 32 tasks an SM on (32 x 148 = 4736); below it, and up to 512 columns, one.
SHAPES = [(5000, 515), (5000, 1000), (2500, 1031), (5000, 1024), (4800, 769), (700, 515), (300, 1031)]


@pytest.mark.parametrize("rows,K", SHAPES)
@pytest.mark.parametrize("G", [32, 64, 128, 256])
@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("scale_dtype", FLOATS)
def test_definition(rows, K, G, dtype, scale_dtype):
    g = torch.Generator(device=DEV).manual_seed(rows + K + G)
    wide = torch.randn(rows, K + 13, generator=g, device=DEV).to(dtype)
    for w in (wide[:, :K].contiguous(), wide[:, 3:3 + K], wide[:, :K]):
        check(w, G, scale_dtype, (dtype,))


def plant(w, G, g):
    """Groups of every kind beside ordinary ones, the same warp's among them."""
    rows, K = w.shape
    groups = (K + G - 1) // G
    kinds = [lambda p: p.zero_(), lambda p: p[:, -1:].fill_(INF), lambda p: p[:, :1].fill_(NAN), lambda p: p[:, :1].fill_(-INF),
             lambda p: p.mul_(2.0 ** -14), lambda p: p.mul_(2.0 ** -20), lambda p: p.mul_(2.0 ** -24), lambda p: p.mul_(2.0 ** 13)]
    if w.dtype is not torch.float16:
        kinds += [lambda p: p.mul_(2.0 ** -105), lambda p: p.mul_(2.0 ** -127), lambda p: p.mul_(2.0 ** -131), lambda p: p.mul_(2.0 ** 110),
                  lambda p: p.mul_(2.0 ** 20)]
    for n in range(rows):
        for e in torch.randint(0, groups, (max(1, groups // 3),), generator=g).tolist():
            kinds[int(torch.randint(0, len(kinds), (1,), generator=g))](w[n:n + 1, e * G:(e + 1) * G])
    return w


@pytest.mark.parametrize("rows,K", [(5000, 1031), (60, 1031), (40, 300)])
@pytest.mark.parametrize("G", [32, 256])
@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("scale_dtype", FLOATS)
def test_special_groups(rows, K, G, dtype, scale_dtype):
    g = torch.Generator().manual_seed(K + G)
    some = plant(torch.randn(60, K, generator=g).to(dtype), G, g)
    at = torch.randint(0, 60, (rows,), generator=g)
    w = some[at].to(DEV)
    for v in (w, torch.cat((w[:, :1], w), 1)[:, 1:]):
        check(v, G, scale_dtype)


@pytest.mark.parametrize("dtype,bits", [(torch.float16, 10), (torch.bfloat16, 7)])
@pytest.mark.parametrize("scale_dtype", FLOATS)
def test_every_quotient_of_16_bits(dtype, bits, scale_dtype):
    """Every mantissa of a group's largest value with every value down to a sixteenth of it, either sign:
    all quotients that round to anything but 0, the halves and those next to halves among them."""
    n = 1 << bits
    top = 1 + torch.arange(n, dtype=torch.float64, device=DEV) / n
    steps = torch.cat([top * 2.0 ** -e for e in range(4, -1, -1)]).to(dtype)     # 1/16 to 2, in order
    tops = top.to(dtype)
    chunks = math.ceil(steps.numel() / 31)
    x = torch.zeros(chunks * 31, dtype=dtype, device=DEV)
    x[:steps.numel()] = steps
    w = torch.empty(n, chunks, 32, dtype=dtype, device=DEV)
    w[..., 0] = tops[:, None]
    w[..., 1:] = torch.where(x.view(1, chunks, 31) <= tops[:, None, None], x.view(1, chunks, 31), 0.0)
    sign = torch.where(torch.rand(w.shape, device=DEV, generator=torch.Generator(device=DEV).manual_seed(1)) < 0.5, -1.0, 1.0)
    w = (w * sign.to(dtype)).view(-1, 32)
    w = w[:w.shape[0] // 32 * 32].reshape(-1, 1024)
    for f in (1.0, 2.0 ** -9, 2.0 ** 12):
        for rows in (*w.split(4000), w.repeat(math.ceil(4800 / w.shape[0]), 1)):      # one span a task, and four
            check((rows * f).to(dtype), 32, scale_dtype, ())
