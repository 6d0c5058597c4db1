"""4-bit weights: quantization against its formula, products against 64 bits.

Bounds of a product: a sum of n fp32 terms is off by at most n units of 2^-23 of the sum of the
terms' sizes (tensor cores may cut where IEEE addition rounds: a whole unit instead of half),
here n = K products, their groups' scalings and additions and the bias; then one rounding to the
type.  With small integers for tokens and powers of two for scales every such sum is a whole
multiple of one power of two below 2^24 of it, so it is exact in any order: the result has to be
the exact value rounded once, bit for bit.
"""
from __future__ import annotations

import pytest
import torch

import metalblas_b200 as mb
from metalblas_b200 import _lib

pytestmark = pytest.mark.gpu
DEV = "cuda"
UNIT = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -24, torch.bfloat16: 2.0 ** -133}
FLOATS = (torch.float32, torch.float16, torch.bfloat16)
TOKENS = (torch.float16, torch.bfloat16)


def gen(seed):
    return torch.Generator().manual_seed(seed)


def weights(lead, K, G, g, scale_dtype, zero, exact=False):
    """Random nibbles, scales and zero points, packed rows on 16-byte boundaries as quantize_int4 makes them."""
    cols, groups = (K + 1) // 2, (K + G - 1) // G
    q = torch.randint(0, 256, (*lead, (cols + 15) // 16 * 16), generator=g, dtype=torch.int32).to(torch.uint8)
    if exact:
        scale = 2.0 ** torch.randint(-2, 2, (*lead, groups), generator=g)
    else:
        scale = torch.rand((*lead, groups), generator=g) * 0.02 + 0.002
    z = torch.randint(0, 16, (*lead, groups), generator=g).to(torch.uint8) if zero else None
    return q.to(DEV)[..., :cols], scale.to(scale_dtype).to(DEV), z.to(DEV) if zero else None


def unpacked(q, scale, zero, K, G):
    """The weights in 64 bits."""
    u = torch.stack((q & 15, q >> 4), -1).reshape(*q.shape[:-1], -1)[..., :K].double()
    at = torch.arange(K, device=q.device) // G
    z = 8.0 if zero is None else zero.double()[..., at]
    return (u - z) * scale.double()[..., at]


def tokens(M, K, g, dtype, exact=False):
    x = torch.randint(-3, 4, (M, K), generator=g).float() if exact else torch.randn(M, K, generator=g)
    return x.to(dtype).to(DEV)


def close(got, want, size, terms):
    u = UNIT[got.dtype]
    tol = terms * 2.0 ** -23 * size * (1 + u) + u * want.abs() + TINY[got.dtype]
    err = (got.double() - want).abs()
    assert bool((err <= tol).all()), f"off by {float((err / tol).max())} of the bound"


# ------------------------------------------------------------------------------ quantize
@pytest.mark.parametrize("shape,G", [((1, 32), 32), ((3, 1), 32), ((5, 33), 32), ((7, 100), 64), ((16, 256), 128),
                                     ((9, 1000), 128), ((4, 4099), 256), ((2, 3, 130), 64), ((130, 512), 256)])
@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("own_scale", [True, False])
def test_quantize(shape, G, dtype, own_scale):
    sd = dtype if own_scale else torch.float32
    w = torch.randn(shape, generator=gen(sum(shape) + G)).to(dtype).to(DEV)
    w.view(-1)[:1] = 0
    K = shape[-1]
    q, s = mb.quantize_int4(w, G, scale_dtype=sd)
    assert q.dtype is torch.uint8 and q.shape == (*shape[:-1], (K + 1) // 2) and s.shape[-1] == (K + G - 1) // G
    assert s.dtype is sd and (len(shape) != 2 or q.stride(0) % 16 == 0 or shape[0] == 1)
    at = torch.arange(K, device=DEV) // G
    amax = torch.zeros((*shape[:-1], s.shape[-1]), dtype=torch.float64, device=DEV)
    amax = amax.scatter_reduce(-1, at.expand(shape), w.double().abs(), "amax")
    assert torch.equal(s, (amax / 7).float().to(sd))
    want = torch.round(w.double() / s.double()[..., at].clamp_min(1e-300)).clamp(-7, 7)
    got = unpacked(q, torch.ones_like(s), None, K, G)
    assert torch.equal(got, want)
    for out in FLOATS:
        back = mb.dequantize_int4(q, s, G, cols=K, out_dtype=out)
        assert back.shape == w.shape and torch.equal(back, (want * s.double()[..., at]).float().to(out))


@pytest.mark.parametrize("dtype", FLOATS)
def test_quantize_halves(dtype):
    """Every quotient n + 1/2: decided to even, also where w / s rounds onto a half in 32 bits."""
    s = 3.0
    w = torch.tensor([[21.0] + [s * (n + 0.5) for n in range(-7, 7)] + [0.0] * 17], device=DEV).to(dtype)
    q, scale = mb.quantize_int4(w, 32)
    assert float(scale) == s
    assert torch.equal(unpacked(q, scale, None, 32, 32), torch.round(w.double() / s) * s)
    # 32-bit neighbours of a half on both sides
    w = torch.tensor([[21.0, 4.5, 4.5 + 2 ** -21, 4.5 - 2 ** -21, -7.5, -7.5 - 2 ** -21, -7.5 + 2 ** -21] + [0.0] * 25],
                     device=DEV)
    q, scale = mb.quantize_int4(w, 32)
    assert unpacked(q, torch.ones_like(scale), None, 32, 32)[0, :7].tolist() == [7, 2, 2, 1, -2, -3, -2]


def test_quantize_special_groups():
    w = torch.randn(4, 128, generator=gen(5)).to(DEV)
    w[0, :32] = 0
    w[1, 3], w[2, 70], w[3, 127] = float("inf"), float("nan"), 2.0 ** -149
    w[3, 96:127] = 0
    q, s = mb.quantize_int4(w, 32)
    u = unpacked(q, torch.ones_like(s), None, 128, 32)
    assert float(s[0, 0]) == 0 and bool((u[0, :32] == 0).all())
    assert bool(s[1, 0].isnan()) and bool((u[1, :32] == 0).all()) and not bool(s[1, 1:].isnan().any())
    assert bool(s[2, 2].isnan()) and bool((u[2, 64:96] == 0).all()) and not bool(u[2, :64].eq(0).all())
    assert float(s[3, 3]) == 0 and bool((u[3, 96:] == 0).all())
    # tiny and huge groups keep their quotients
    for f in (2.0 ** -130, 2.0 ** 120):
        w = torch.tensor([[7.0, 3.4, -6.6, 0.2] + [0.0] * 28], device=DEV) * f
        q, s = mb.quantize_int4(w, 32)
        assert unpacked(q, torch.ones_like(s), None, 32, 32)[0, :4].tolist() == [7, 3, -7, 0]


def test_quantize_strided_rows_and_zero_points():
    w = torch.randn(40, 300, generator=gen(6)).to(DEV)
    for v in (w[:, 1:-3], w[::2], w.t(), w[3:4].expand(5, 300)):
        a, b = mb.quantize_int4(v, 64), mb.quantize_int4(v.contiguous(), 64)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    q, s, z = weights((6, 5), 77, 32, gen(7), torch.float16, True)
    want = unpacked(q, s, z, 77, 32)
    for out in FLOATS:
        assert torch.equal(mb.dequantize_int4(q, s, 32, zero=z, cols=77, out_dtype=out), want.float().to(out))


# ------------------------------------------------------------------------------ products
SHAPES = [(1, 32, 1, 32), (1, 64, 64, 64), (1, 4096, 512, 128), (1, 1, 5, 32), (2, 100, 33, 32), (3, 4099, 130, 128),
          (4, 1000, 77, 256), (5, 2051, 300, 64), (7, 256, 16, 128), (8, 1024, 1000, 32), (9, 515, 129, 64),
          (13, 8192, 48, 128), (16, 2048, 256, 256), (17, 384, 200, 128), (31, 130, 31, 32), (32, 640, 512, 64),
          (33, 1025, 127, 128), (64, 4096, 384, 128), (100, 260, 140, 32), (129, 999, 257, 256), (255, 512, 640, 128),
          (300, 2000, 130, 64), (520, 1152, 384, 128)]


@pytest.mark.parametrize("M,K,N,G", SHAPES)
@pytest.mark.parametrize("dtype", TOKENS)
@pytest.mark.parametrize("zero", [False, True])
def test_product(M, K, N, G, dtype, zero):
    g = gen(M * 7 + K + N)
    for exact in (True, False):
        sd = dtype if zero else torch.float32
        q, s, z = weights((N,), K, G, g, sd, zero, exact)
        x = tokens(M, K, g, dtype, exact)
        w = unpacked(q, s, z, K, G)
        want = x.double() @ w.t()
        got = mb.int4_mm(x, q, s, G, zero=z)
        assert got.dtype is dtype
        if exact:
            assert torch.equal(got, want.to(dtype))
        bias = torch.randn(N, generator=g).to(dtype if zero else torch.float32).to(DEV)
        size = x.double().abs() @ w.abs().t()
        close(got, want, size, K + 2 * s.shape[1])
        close(mb.int4_mm(x, q, s, G, zero=z, bias=bias), want + bias.double(), size + bias.double().abs(),
              K + 2 * s.shape[1] + 1)


def split(counts):
    off = [0]
    for c in counts:
        off.append(off[-1] + c)
    return torch.tensor(off, dtype=torch.int32, device=DEV)


GROUPED = [([1], 0, 64, 64, 32), ([0, 3, 0, 1], 2, 100, 33, 64), ([2, 2, 2, 2, 1, 0, 1, 3], 0, 1024, 130, 128),
           ([5, 0, 9, 16, 17, 1], 3, 515, 200, 32), ([0, 0, 0], 4, 64, 16, 64), ([40, 1, 200, 0, 33], 7, 384, 257, 128),
           ([130, 129, 300, 2], 1, 1000, 384, 256), ([8] * 20 + [0] * 20, 0, 256, 96, 128),
           ([1, 0, 2, 0] * 30, 5, 130, 72, 64)]


@pytest.mark.parametrize("counts,rest,K,N,G", GROUPED)
@pytest.mark.parametrize("dtype", TOKENS)
@pytest.mark.parametrize("zero", [False, True])
def test_grouped_product(counts, rest, K, N, G, dtype, zero):
    g = gen(sum(counts) + K + N)
    E, M = len(counts), sum(counts) + rest
    off = split(counts)
    for exact in (True, False):
        q, s, z = weights((E, N), K, G, g, torch.float32 if zero else dtype, zero, exact)
        x = tokens(M, K, g, dtype, exact)
        x[sum(counts):] = float("nan")    # rows of no group are not read
        w = unpacked(q, s, z, K, G)
        want = torch.zeros((M, N), dtype=torch.float64, device=DEV)
        size = torch.zeros_like(want)
        for e, c in enumerate(counts):
            a, b = int(off[e]), int(off[e + 1])
            want[a:b] = x[a:b].double() @ w[e].t()
            size[a:b] = x[a:b].double().abs() @ w[e].abs().t()
        got = mb.grouped_int4_mm(x, q, s, off, G, zero=z)
        assert bool((got[sum(counts):] == 0).all())
        if exact:
            assert torch.equal(got, want.to(dtype))
        close(got, want, size, K + 2 * s.shape[-1])


def test_offsets_that_name_no_groups():
    q, s, _ = weights((3, 40), 64, 32, gen(1), torch.float32, False)
    x = tokens(12, 64, gen(2), torch.bfloat16)
    for off in ([0, 8, 4, 12], [0, 4, 8, 7]):
        got = mb.grouped_int4_mm(x, q, s, torch.tensor(off, dtype=torch.int32, device=DEV), 32)
        assert bool((got == 0).all())
    # numbers outside 0..M are the nearest of the two
    got = mb.grouped_int4_mm(x, q, s, torch.tensor([-5, 4, 8, 99], dtype=torch.int32, device=DEV), 32)
    assert torch.equal(got, mb.grouped_int4_mm(x, q, s, split([4, 4, 4]), 32))


@pytest.mark.parametrize("M", [1, 6, 40])
def test_no_columns_and_empty(M):
    x = torch.zeros(M, 0, dtype=torch.bfloat16, device=DEV)
    q, s = torch.zeros(8, 0, dtype=torch.uint8, device=DEV), torch.zeros(8, 0, device=DEV)
    b = torch.arange(8, device=DEV).bfloat16()
    assert bool((mb.int4_mm(x, q, s) == 0).all()) and torch.equal(mb.int4_mm(x, q, s, bias=b), b.expand(M, 8))
    q, s, _ = weights((8,), 64, 32, gen(3), torch.float32, False)
    assert mb.int4_mm(x.new_zeros(0, 64), q, s, 32).shape == (0, 8)
    assert mb.int4_mm(x.new_zeros(M, 64), q[:0], s[:0], 32).shape == (M, 0)
    assert mb.int4_mm(x.new_zeros(2, 3, 64), q, s, 32).shape == (2, 3, 8)
    assert mb.int4_mm(x.new_zeros(64), q, s, 32).shape == (8,)


@pytest.mark.parametrize("M", [1, 12, 50])
def test_layouts(M):
    """Strides, offsets and orders of every operand give the bits of the plain layout."""
    K, N, G = 328, 90, 64
    g = gen(9)
    q, s, z = weights((N,), K, G, g, torch.bfloat16, True)
    x = tokens(M, K, g, torch.bfloat16)
    want = mb.int4_mm(x, q, s, G, zero=z)
    wide = torch.zeros(M, K + 40, dtype=x.dtype, device=DEV)
    for at in (0, 1, 8):
        wide[:, at:at + K] = x
        assert torch.equal(mb.int4_mm(wide[:, at:at + K], q, s, G, zero=z), want)
    assert torch.equal(mb.int4_mm(x.t().contiguous().t(), q, s, G, zero=z), want)
    tight = q.contiguous()                                  # 164 bytes a row
    assert torch.equal(mb.int4_mm(x, tight, s, G, zero=z), want)
    off = torch.zeros(N * 164 + 1, dtype=torch.uint8, device=DEV)
    off[1:] = tight.reshape(-1)
    assert torch.equal(mb.int4_mm(x, off[1:].view(N, 164), s.t().contiguous().t(), G, zero=z.t().contiguous().t()), want)
    twice = torch.stack((q, q), 1).reshape(2 * N, -1)[::2]
    assert torch.equal(mb.int4_mm(x, twice, torch.stack((s, s), 1)[:, 0], G, zero=z), want)
    buf = torch.full((M + 2, N + 5), 7.0, dtype=x.dtype, device=DEV)
    mb.int4_mm(x, q, s, G, zero=z, out=buf[1:M + 1, 3:N + 3])
    assert torch.equal(buf[1:M + 1, 3:N + 3], want)
    buf[1:M + 1, 3:N + 3] = 7.0
    assert bool((buf == 7.0).all())                          # nothing beside the result is written


@pytest.mark.parametrize("M", [3, 60])
def test_non_finite_tokens(M):
    """An infinity or a NaN reaches its own row alone; columns past K are not read."""
    K, N, G = 70, 40, 32
    q, s, _ = weights((N,), K, G, gen(4), torch.float32, False)
    full = torch.full((M, K + 26), float("nan"), dtype=torch.float16, device=DEV)
    full[:, :K] = tokens(M, K, gen(5), torch.float16)
    want = mb.int4_mm(full[:, :K].contiguous(), q, s, G)
    assert bool(want.isfinite().all()) and torch.equal(mb.int4_mm(full[:, :K], q, s, G), want)
    full[1, 5], full[2, 6] = float("nan"), float("inf")
    got = mb.int4_mm(full[:, :K], q, s, G)
    assert bool(got[1].isnan().all()) and not bool(got[2].isfinite().any())
    keep = [m for m in range(M) if m not in (1, 2)]
    assert torch.equal(got[keep], want[keep])


def test_refusals():
    q, s, z = weights((8,), 64, 32, gen(3), torch.bfloat16, True)
    x = tokens(2, 64, gen(4), torch.bfloat16)
    cases = [
        (lambda: mb.int4_mm(x.float(), q, s, 32), NotImplementedError),
        (lambda: mb.int4_mm(x, q, s.half(), 32), NotImplementedError),
        (lambda: mb.int4_mm(x, q.to(torch.int8), s, 32), NotImplementedError),
        (lambda: mb.int4_mm(x, q, s, 32, zero=z.float()), NotImplementedError),
        (lambda: mb.int4_mm(x, q, s, 48), ValueError),
        (lambda: mb.int4_mm(x, q, s, 64), AssertionError),
        (lambda: mb.int4_mm(x[:, :60], q, s, 32), AssertionError),
        (lambda: mb.int4_mm(x, q, s, 32, zero=z[:4]), AssertionError),
        (lambda: mb.int4_mm(x, q, s, 32, bias=s[0]), AssertionError),
        (lambda: mb.int4_mm(x, q, s.cpu(), 32), AssertionError),
        (lambda: mb.int4_mm(x, q, 1.0, 32), AssertionError),
        (lambda: mb.int4_mm(x, q, s, 32, out=torch.empty(2, 8, device=DEV)), ValueError),
        (lambda: mb.int4_mm(x, q, s, 32, out=torch.empty(8, 2, device=DEV, dtype=x.dtype).t()), AssertionError),
        (lambda: mb.int4_mm(x, q, s, 32, out=torch.empty(1, 8, device=DEV, dtype=x.dtype).expand(2, 8)), ValueError),
        (lambda: mb.int4_mm(x.clone().requires_grad_(), q, s, 32), NotImplementedError),
        (lambda: mb.grouped_int4_mm(x, q[None], s[None], torch.tensor([0, 2], device=DEV), 32), NotImplementedError),
        (lambda: mb.grouped_int4_mm(x, q[None], s[None], split([1, 1]), 32), AssertionError),
        (lambda: mb.quantize_int4(x, 16), ValueError),
        (lambda: mb.quantize_int4(x.double()), NotImplementedError),
        (lambda: mb.dequantize_int4(q, s, 32, cols=62), AssertionError),
    ]
    for i, (call, error) in enumerate(cases):
        with pytest.raises(error):
            call()
            pytest.fail(f"case {i} was not refused")
    with torch.no_grad():
        mb.int4_mm(x.clone().requires_grad_(), q, s, 32)


@pytest.mark.parametrize("M", [2, 48])
def test_capture_and_streams(M):
    """Two captured calls replayed on another stream, after inputs changed in place."""
    K, N, G = 1024, 256, 128
    q, s, z = weights((N,), K, G, gen(11), torch.bfloat16, True)
    x = tokens(M, K, gen(12), torch.bfloat16)
    off = split([M // 2, M - M // 2])
    q2, s2, _ = weights((2, N), K, G, gen(13), torch.float32, False)
    call = lambda: (mb.int4_mm(x, q, s, G, zero=z), mb.grouped_int4_mm(x, q2, s2, off, G))
    call()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    x.copy_(tokens(M, K, gen(14), torch.bfloat16))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        graph.replay()
        plain = call()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(out, plain))
    assert _lib.device_status() == 0
