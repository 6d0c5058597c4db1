"""int8 rows and the int8 products with scales, against the formulas in 64 bits.

The products' sums are exact, so the only roundings are the sum's conversion to fp32, two
products with scales and the bias sum in fp32 (each at most 2^-24 of its result), and the
rounding to the output's type; the tolerances below are those, added up.
"""
from __future__ import annotations

import pytest
import torch

import metalblas_b200 as mb
from metalblas_b200 import kernels

pytestmark = pytest.mark.gpu
DEV = "cuda"
FLOATS = (torch.float32, torch.float16, torch.bfloat16)
U32 = 2.0 ** -24
UNIT = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -24, torch.bfloat16: 2.0 ** -133}


@pytest.fixture(autouse=True)
def no_wait_gave_up():
    yield
    assert kernels.device_status() == 0


def gen(seed):
    return torch.Generator().manual_seed(seed)


def ints(shape, g):
    return torch.randint(-127, 128, shape, dtype=torch.int8, generator=g).to(DEV)


def scales(shape, g):
    return (torch.rand(shape, generator=g) * 0.02 + 1e-3).to(DEV)


# ------------------------------------------------------------------------------ quantize
def plain_quantize(x):
    xd = x.double()
    amax = xd.abs().amax(-1, keepdim=True)
    q = torch.where(amax > 0, xd * 127 / torch.where(amax > 0, amax, 1.0), torch.zeros_like(xd)).round()
    return q.to(torch.int8), (amax[..., 0] / 127)


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 7), (3, 16), (5, 33), (17, 129), (2, 2048), (64, 4096), (7, 4100),
                                       (3, 16384), (2, 40000), (1000, 64), (1, 100001), (4099, 4096), (4096, 2056),
                                       (600, 14336), (300, 1000), (70, 8200)])
def test_quantize_is_the_formula(rows, cols, dtype):
    x = torch.randn(rows, cols, generator=gen(rows + cols)).to(dtype).to(DEV)
    q, s = mb.quantize(x)
    want, ws = plain_quantize(x)
    assert q.dtype is torch.int8 and s.dtype is torch.float32 and q.shape == x.shape and s.shape == (rows,)
    if dtype is torch.float32:
        # 127 x is rounded: a quotient within 2^-22 of a half may go either way
        d = x.double() * 127 / x.double().abs().amax(-1, keepdim=True)
        near = ((d - d.floor()) - 0.5).abs() < 127 * 2.0 ** -22
        assert bool(((q == want) | near).all()) and int((q.int() - want.int()).abs().max()) <= 1
    else:
        assert torch.equal(q, want)
    assert bool(((s.double() - ws).abs() <= U32 * ws).all())


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_quantize_rounds_halves_to_even(dtype):
    """amax = 127 or 254 puts halves exactly where they are in the formula."""
    x = torch.arange(-254, 255, dtype=torch.float32)
    x = torch.stack([x, x / 2, x * 2.0 ** -9]).to(dtype).to(DEV)
    assert torch.equal(mb.quantize(x)[0], plain_quantize(x)[0])


def test_every_bf16_ratio_is_the_formula():
    """All pairs of 8-bit significands as (x, amax)."""
    m = torch.arange(128, 256, dtype=torch.float32)
    x = torch.cat([m[None, :].expand(128, 128), m[None, :].expand(128, 128) / 4, m[None, :].expand(128, 128) / 32], 1)
    x = torch.cat([torch.minimum(x, m[:, None] * 2), m[:, None] * 2], 1).to(torch.bfloat16).to(DEV)
    assert torch.equal(mb.quantize(x)[0], plain_quantize(x)[0])


@pytest.mark.parametrize("dtype", FLOATS)
def test_quantize_special_rows(dtype):
    f = torch.finfo(dtype)
    x = torch.randn(8, 40, generator=gen(3)).to(dtype)
    x[0] = 0
    x[1, 5] = float("inf")
    x[2, 6] = float("nan")
    x[3, 7] = -float("inf")
    x[4] = 0
    x[4, 0], x[4, 1], x[4, 2] = f.max, f.min, f.max / 2
    x[5] = 0
    x[5, 39], x[5, 0] = f.tiny, -f.tiny / 2
    x[6] = -0.0
    x = x.to(DEV)
    q, s = mb.quantize(x)
    q, s = q.cpu(), s.cpu()
    assert bool((q[[0, 1, 2, 3, 6]] == 0).all())
    assert s[0] == 0 and s[6] == 0 and bool(torch.isnan(s[1:4]).all())
    for r in (4, 5, 7):
        want, ws = plain_quantize(x[r:r + 1].cpu())
        assert torch.equal(q[r:r + 1], want)
        assert abs(float(s[r]) - float(ws)) <= U32 * float(ws) + 2.0 ** -150


def test_quantize_layouts():
    g = gen(5)
    base = torch.randn(40, 200, generator=g).to(torch.bfloat16).to(DEV)
    for x in (base[:, 3:70], base[::2], base[1:, 8:136], base.t(), base.expand(3, 40, 200), base.view(2, 20, 200),
              base[0], base[:0], base[:1, :17], base[:, :0]):
        q, s = mb.quantize(x)
        assert q.shape == x.shape and s.shape == x.shape[:-1]
        if x.numel():
            want, ws = plain_quantize(x)
            assert torch.equal(q, want)
            assert bool(((s.double() - ws).abs() <= U32 * ws).all())
        else:
            assert bool((s == 0).all())


# ------------------------------------------------------------------------------ products
def check_product(y, q, w, sa, sb, bias=None):
    """y against the 64-bit formula, within the roundings named above."""
    p = (q.double() @ w.double()) * sa.double()[:, None] * sb.double()
    want = p if bias is None else p + bias.double()
    size = p.abs() + (0 if bias is None else bias.double().abs())
    u = UNIT[y.dtype]
    tol = 4 * U32 * size * (1 + u) + u * want.abs() + TINY[y.dtype]
    bad = (y.double() - want).abs() > tol
    assert not bool(bad.any()), f"{int(bad.sum())} of {bad.numel()} values off"


SHAPES = [(1, 1, 1), (1, 16, 16), (1, 4096, 512), (2, 33, 77), (3, 128, 128), (5, 4096, 640), (16, 1024, 2048),
          (17, 48, 31), (33, 256, 4099), (64, 512, 1000), (100, 4100, 260), (128, 128, 128), (129, 272, 257),
          (200, 1008, 515), (300, 64, 2051), (513, 2048, 768), (1000, 513, 130)]


@pytest.mark.parametrize("M,K,N", SHAPES)
@pytest.mark.parametrize("layout", ["nk", "kn"])
def test_scaled_mm(M, K, N, layout):
    g = gen(M * 7 + K + N)
    a, sa, sb = ints((M, K), g), scales((M,), g), scales((N,), g)
    w = ints((N, K), g).t() if layout == "nk" else ints((K, N), g)
    for out_dtype in FLOATS:
        y = mb.scaled_mm(a, w, sa, sb, out_dtype=out_dtype)
        assert y.dtype is out_dtype and y.shape == (M, N)
        check_product(y, a, w, sa, sb)


@pytest.mark.parametrize("M,K,N", [(1, 64, 48), (5, 96, 33), (40, 1024, 300), (150, 128, 257), (260, 272, 515)])
@pytest.mark.parametrize("out_dtype", FLOATS)
def test_scaled_mm_bias(M, K, N, out_dtype):
    g = gen(M + K + N)
    a, w, sa, sb = ints((M, K), g), ints((N, K), g).t(), scales((M,), g) , scales((N,), g)
    for bias_dtype in {out_dtype, torch.float32}:
        for bias in (torch.randn(N, generator=g).to(bias_dtype).to(DEV),
                     torch.randn(2 * N, generator=g).to(bias_dtype).to(DEV)[::2]):
            y = mb.scaled_mm(a, w, sa, sb, bias=bias, out_dtype=out_dtype)
            check_product(y, a, w, sa, sb, bias)


@pytest.mark.parametrize("M", [1, 2, 3, 7, 8, 9, 15, 16, 17])
@pytest.mark.parametrize("K", [1, 15, 16, 63, 65, 500, 1040, 2050])
def test_scaled_mm_few_rows(M, K):
    """The single-pass kernels: rows of K bytes in aligned storage, few and many channels."""
    g = gen(M * 3 + K)
    room = (K + 15) // 16 * 16 + 32
    A = ints((M, room), g)[:, :K]
    for N in (1, 5, 148, 297, 2000, 40000 if K > 1000 else 601):
        w, sa, sb = ints((N, room), g)[:, :K].t(), scales((M,), g), scales((N,), g)
        bias = torch.randn(N, generator=g).to(DEV)
        for out_dtype in (torch.bfloat16, torch.float32):
            y = mb.scaled_mm(A, w, sa, sb, bias=bias if N % 2 else None, out_dtype=out_dtype)
            check_product(y, A, w, sa, sb, bias if N % 2 else None)
        assert torch.equal(y, mb.scaled_mm(A, w, sa, sb, bias=bias if N % 2 else None, out_dtype=torch.float32,
                                           _plan=(16, 1, 1, 1)))


def test_scaled_mm_extreme_values_are_exact():
    """The longest K of -128 * -128 and -128 * 127: no sum wraps."""
    K = 131071
    a = torch.full((2, K), -128, dtype=torch.int8, device=DEV)
    w = torch.full((8, K), -128, dtype=torch.int8, device=DEV)
    w[1] = 127
    y = mb.scaled_mm(a, w.t(), torch.ones(2, device=DEV), torch.ones(8, device=DEV), out_dtype=torch.float32)
    assert float(y[0, 0]) == float(torch.tensor(K * 16384, dtype=torch.int64).float())
    assert float(y[1, 1]) == float(torch.tensor(-K * 128 * 127, dtype=torch.int64).float())


def test_scaled_mm_layouts_and_out():
    g = gen(11)
    A, W = ints((80, 400), g), ints((300, 400), g)
    sa, sb = scales((80,), g), scales((300,), g)
    for a in (A, A.t().contiguous().t(), A[:, 1:301], A[::2, :200], A[3:, 16:272]):
        M, K = a.shape
        for w in (W[:, :K].t(), W.t()[:K], W[:, :K].t().contiguous(), W[::2, 1:K + 1].t() if K < 400 else W[::2].t(),
                  W[:, :K].t()[:, 5:70], ints((K, 600), g)[:, ::2]):
            N = w.shape[1]
            y = mb.scaled_mm(a, w, sa[:M], sb[:N], out_dtype=torch.float32)
            check_product(y, a, w, sa[:M], sb[:N])
    w = W.t()
    for out in (torch.empty(300, 80, device=DEV).t(), torch.empty(80, 333, device=DEV)[:, 7:307],
                torch.empty(160, 600, device=DEV)[::2, ::2]):
        r = mb.scaled_mm(A, w, sa, sb, out=out)
        assert r.data_ptr() == out.data_ptr()
        check_product(out, A, w, sa, sb)
    wide = torch.full((80, 333), 7.0, device=DEV)
    mb.scaled_mm(A, w, sa, sb, out=wide[:, 7:307])
    assert bool((wide[:, :7] == 7).all()) and bool((wide[:, 307:] == 7).all())
    a3 = A.view(4, 20, 400)
    y = mb.scaled_mm(a3, w, sa.view(4, 20), sb, out_dtype=torch.float32)
    assert y.shape == (4, 20, 300)
    check_product(y.view(80, 300), A, w, sa, sb)
    y = mb.scaled_mm(A[0], w, sa[0], sb, out_dtype=torch.float32)
    assert y.shape == (300,)
    check_product(y[None], A[:1], w, sa[:1], sb)


def test_scaled_mm_broadcast_scales():
    g = gen(12)
    a, w = ints((37, 64), g), ints((50, 64), g).t()
    sa, sb = scales((37,), g), scales((50,), g)
    one = scales((), g)
    check_product(mb.scaled_mm(a, w, one, sb, out_dtype=torch.float32), a, w, one.expand(37), sb)
    check_product(mb.scaled_mm(a, w, sa, one.reshape(1), out_dtype=torch.float32), a, w, sa, one.expand(50))
    two = torch.stack([sa, sa], 1)[:, 0]
    check_product(mb.scaled_mm(a, w, two, sb, out_dtype=torch.float32), a, w, sa, sb)


def test_scaled_mm_empty():
    g = gen(13)
    z = lambda *s: torch.zeros(*s, dtype=torch.int8, device=DEV)  # noqa: E731
    assert mb.scaled_mm(z(0, 8), z(8, 5), scales((0,), g), scales((5,), g)).shape == (0, 5)
    assert mb.scaled_mm(z(4, 8), z(8, 0), scales((4,), g), scales((0,), g)).shape == (4, 0)
    bias = torch.randn(5, generator=g).to(DEV)
    y = mb.scaled_mm(z(4, 0), z(0, 5), scales((4,), g), scales((5,), g), bias=bias, out_dtype=torch.float32)
    assert torch.equal(y, bias.expand(4, 5))


def test_scaled_mm_carries_non_finite_scales():
    g = gen(14)
    x = torch.randn(130, 64, generator=g)
    x[3, 5], x[128, 0] = float("nan"), float("inf")
    x[7] = 0
    q, s = mb.quantize(x.to(DEV))
    w, sb = ints((40, 64), g).t(), scales((40,), g)
    for rows in (slice(0, 130), slice(0, 8)):
        y = mb.scaled_mm(q[rows], w, s[rows], sb)
        nan = torch.isnan(y).all(1).cpu()
        bad = torch.isnan(y).any(1).cpu()
        assert torch.equal(nan, bad)
        assert [i for i in range(nan.numel()) if nan[i]] == ([3, 128] if nan.numel() > 128 else [3])
        assert bool((y[7] == 0).all())


def test_scaled_mm_does_not_depend_on_the_batch():
    """The same token gives the same bits alone, among few and among many."""
    g = gen(15)
    a, w, sa, sb = ints((300, 1040), g), ints((500, 1040), g).t(), scales((300,), g), scales((500,), g)
    whole = mb.scaled_mm(a, w, sa, sb)
    for m in (1, 2, 7, 16, 33, 64, 100, 128, 200):
        assert torch.equal(mb.scaled_mm(a[:m], w, sa[:m], sb), whole[:m])


# ------------------------------------------------------------------------------ grouped
def offsets_of(counts):
    return torch.tensor([0] + list(torch.tensor(counts).cumsum(0)), dtype=torch.int32, device=DEV)


def check_grouped(y, a, w, sa, sb, offsets):
    ends = offsets.tolist()
    for e in range(len(ends) - 1):
        r = slice(ends[e], ends[e + 1])
        if ends[e + 1] > ends[e]:
            check_product(y[r], a[r], w[e], sa[r], sb[e])
    assert bool((y[ends[-1]:] == 0).all())


GROUPS = [([1], 0), ([0, 0, 3], 0), ([0], 4), ([0, 0], 0), ([5, 0, 1, 16, 17, 0], 3), ([128, 1, 127, 129], 0), ([300, 0, 40], 50),
          ([1] * 40, 0), ([2, 0] * 32, 1), ([64, 63, 65, 33], 130), ([700], 1)]


@pytest.mark.parametrize("counts,extra", GROUPS)
@pytest.mark.parametrize("K,N", [(64, 48), (128, 128), (272, 390), (1040, 256), (100, 33)])
def test_grouped(counts, extra, K, N):
    g = gen(sum(counts) + K + N + extra)
    M, E = sum(counts) + extra, len(counts)
    a, sa, sb = ints((M, K), g), scales((M,), g), scales((E, N), g)
    off = offsets_of(counts)
    for w in (ints((E, N, K), g).transpose(1, 2), ints((E, K, N), g)):
        for out_dtype in FLOATS:
            y = mb.grouped_scaled_mm(a, w, sa, sb, off, out_dtype=out_dtype,
                                     out=torch.full((M, N), float("nan"), dtype=out_dtype, device=DEV))
            check_grouped(y, a, w, sa, sb, off)


def test_grouped_many_experts():
    g = gen(21)
    counts = torch.randint(0, 4, (1024,), generator=g).tolist()
    M, K, N = sum(counts), 64, 32
    a, w = ints((M, K), g), ints((1024, N, K), g).transpose(1, 2)
    sa, sb, off = scales((M,), g), scales((1024, N), g), offsets_of(counts)
    check_grouped(mb.grouped_scaled_mm(a, w, sa, sb, off, out_dtype=torch.float32), a, w, sa, sb, off)


@pytest.mark.parametrize("K", [1, 17, 432, 512, 513, 1024, 1040, 2047, 2048, 2064])
def test_few_rows_of_short_sums(K):
    """More weight rows than warps: short rows are taken whole, several at a time."""
    g = gen(K)
    room = (K + 15) // 16 * 16
    for N in (4800, 9473, 40001):
        W, sb = ints((N, room), g)[:, :K].t(), scales((N,), g)
        for M in (1, 2):
            a, sa = ints((M, room), g)[:, :K], scales((M,), g)
            check_product(mb.scaled_mm(a, W, sa, sb, out_dtype=torch.float32), a, W, sa, sb)
    for counts, N in (([2, 0, 1], 1601), ([1, 1, 0, 3, 1, 1, 1], 613), ([0, 5], 3001)):
        M = sum(counts)
        W, sb = ints((len(counts), N, room), g)[:, :, :K].transpose(1, 2), scales((len(counts), N), g)
        for extra in (0, 1):
            if M + extra > 8:
                continue
            a, sa = ints((M + extra, room), g)[:, :K], scales((M + extra,), g)
            y = mb.grouped_scaled_mm(a, W, sa, sb, offsets_of(counts), out_dtype=torch.float32)
            check_grouped(y, a, W, sa, sb, offsets_of(counts))


@pytest.mark.parametrize("K", [63, 700])
def test_grouped_weights_off_16_bytes_few_used(K):
    """Weights copied first, of the groups with rows alone: every group's place in turn."""
    g = gen(K)
    E, N = 600, 33
    for layout in ("nk", "kn"):
        W = ints((E, N, K), g).transpose(1, 2) if layout == "nk" else ints((E, K, N), g)
        sb = scales((E, N), g)
        for used in ([0], [599], [255, 256], list(range(0, 600, 7)), [3, 400, 599]):
            counts = [0] * E
            for i, e in enumerate(used):
                counts[e] = 1 + i % 3
            M = sum(counts)
            a, sa, off = ints((M, K), g), scales((M,), g), offsets_of(counts)
            check_grouped(mb.grouped_scaled_mm(a, W, sa, sb, off, out_dtype=torch.float32), a, W, sa, sb, off)


@pytest.mark.parametrize("out_dtype", FLOATS)
def test_rows_of_the_output_that_start_anywhere(out_dtype):
    """Every start of a row against 16 bytes, every end; what lies around the rows stays."""
    g = gen(31)
    M, K = 150, 64
    a, sa = ints((M, K), g), scales((M,), g)
    off = offsets_of([70, 0, 45, 30])  # and five rows of no group
    for N in (31, 32, 33, 63, 64, 100, 128, 129, 161, 255, 257, 300, 523):
        w, sb = ints((N, K), g).t(), scales((N,), g)
        W, SB = ints((4, N, K), g).transpose(1, 2), scales((4, N), g)
        for start, pitch in ((0, N + 9), (1, N + 1), (3, N + 7), (4, N + 8), (6, N + 13), (7, N + 26)):
            for plan in ((128, 1, -1, 1), (256, 1, -1, 1), (256, 1, -1, 2), (64, 1, 1, 1)):
                room = torch.full((M + 1, pitch), 7.0, dtype=out_dtype, device=DEV).view(-1)
                view = room[start:start + (M - 1) * pitch + N].as_strided((M, N), (pitch, 1), start)
                kept = room.clone()
                kept.as_strided((M, N), (pitch, 1), start).fill_(0)
                mb.scaled_mm(a, w, sa, sb, out=view, _plan=plan)
                check_product(view, a, w, sa, sb)
                view_copy = room.clone()
                view_copy.as_strided((M, N), (pitch, 1), start).fill_(0)
                assert torch.equal(view_copy, kept)
                mb.grouped_scaled_mm(a, W, sa, SB, off, out=view, _plan=plan)
                check_grouped(view, a, W, sa, SB, off)
                view_copy = room.clone()
                view_copy.as_strided((M, N), (pitch, 1), start).fill_(0)
                assert torch.equal(view_copy, kept)


def test_grouped_strides_and_broadcast_scales():
    g = gen(22)
    counts = [20, 0, 33]
    M, K, N, E = 53, 160, 96, 3
    a = ints((M, 2 * K), g)[:, K:]
    W = ints((2 * E, N, K + 32), g)
    off = offsets_of(counts)
    sa, sb = scales((M,), g), scales((E, N), g)
    for w in (W[::2, :, :K].transpose(1, 2), W[:E, :, 32:].transpose(1, 2), W[:E, :, 1:K + 1].transpose(1, 2)):
        y = mb.grouped_scaled_mm(a, w, sa, sb, off, out_dtype=torch.float32)
        check_grouped(y, a, w, sa, sb, off)
    w = W[:1, :, :K].transpose(1, 2).expand(E, K, N)  # one weight for every group
    one = scales((1,), g)
    y = mb.grouped_scaled_mm(a, w, one, sb[:, :1], off, out_dtype=torch.float32)
    check_grouped(y, a, w, one.expand(M), sb[:, :1].expand(E, N), off)
    out = torch.full((M, 2 * N), 5.0, device=DEV)
    mb.grouped_scaled_mm(a, w, sa, sb, off, out=out[:, N:])
    check_grouped(out[:, N:], a, w, sa, sb, off)
    assert bool((out[:, :N] == 5).all())


def test_grouped_offsets_outside_the_rows_stay_inside():
    """Row numbers past the end are taken as the end; nothing outside out is touched."""
    g = gen(23)
    M, K, N = 40, 64, 64
    a, w, sa, sb = ints((M, K), g), ints((2, N, K), g).transpose(1, 2), scales((M,), g), scales((2, N), g)
    off = torch.tensor([0, 30, 1000], dtype=torch.int32, device=DEV)
    room = torch.full((M + 8, N), 9.0, device=DEV)
    mb.grouped_scaled_mm(a, w, sa, sb, off, out=room[:M])
    check_grouped(room[:M], a, w, sa, sb, torch.tensor([0, 30, 40]))
    assert bool((room[M:] == 9).all())


@pytest.mark.parametrize("M", [6, 40, 700])
def test_grouped_offsets_that_are_not_ascending_name_no_groups(M):
    g = gen(26)
    K, N = 64, 80
    a, w, sa, sb = ints((M, K), g), ints((4, N, K), g).transpose(1, 2), scales((M,), g), scales((4, N), g)
    for off in ([0, M, 0, M, 2], [0, 5, 3, M, M], [0, -1 << 31, M, (1 << 31) - 1, 1]):
        off = torch.tensor(off, dtype=torch.int32, device=DEV)
        y = mb.grouped_scaled_mm(a, w, sa, sb, off, out=torch.full((M, N), 3.0, device=DEV))
        assert bool((y == 0).all())


def test_grouped_equals_dense():
    g = gen(24)
    counts = [70, 3, 200]
    M, K, N = 273, 528, 300
    a, W, sa, sb = ints((M, K), g), ints((3, N, K), g), scales((M,), g), scales((3, N), g)
    y = mb.grouped_scaled_mm(a, W.transpose(1, 2), sa, sb, offsets_of(counts))
    at = 0
    for e, c in enumerate(counts):
        r = slice(at, at + c)
        assert torch.equal(y[r], mb.scaled_mm(a[r], W[e].t(), sa[r], sb[e]))
        at += c


def test_on_another_stream_and_in_a_graph():
    g = gen(25)
    x = torch.randn(24, 256, generator=g).to(torch.bfloat16).to(DEV)
    w, sb = ints((512, 256), g).t(), scales((512,), g)
    torch.cuda.synchronize()
    st = torch.cuda.Stream()
    with torch.cuda.stream(st):
        q, s = mb.quantize(x)
        y = mb.scaled_mm(q, w, s, sb)
    st.synchronize()
    q0, s0 = mb.quantize(x)
    y0 = mb.scaled_mm(q0, w, s0, sb)
    assert torch.equal(y, y0)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        q1, s1 = mb.quantize(x)
        y1 = mb.scaled_mm(q1, w, s1, sb)
    x.copy_(torch.randn(24, 256, generator=g).to(torch.bfloat16))
    graph.replay()
    q0, s0 = mb.quantize(x)
    assert torch.equal(y1, mb.scaled_mm(q0, w, s0, sb))


# ------------------------------------------------------------------------------ every plan
PLANS = [(bn, split, 1, 0) for bn in (16, 32, 64, 128) for split in (1, 2, 4, 8)] + \
        [(128, split, -1, 0) for split in (1, 2, 4, 8)] + [(256, 0, -1, 1), (256, 0, -1, 2)]


@pytest.mark.parametrize("plan", PLANS)
def test_every_tile_and_split_gives_the_same_bits(plan):
    """(tile_n, split, swap, pair) as given, over ragged tiles and, for the splits, more units
    than clusters, so that each cluster hands its partial sums over several times."""
    g = gen(41)
    for M, K, N in ((1, 1040, 260), (130, 1040, 515), (300, 1296, 1000), (40, 1024, 30000)):
        a, sa, sb = ints((M, K), g), scales((M,), g), scales((N,), g)
        bias = torch.randn(N, generator=g).to(DEV)
        for w in (ints((N, K), g).t(), ints((K, (N + 15) // 16 * 16), g)[:, :N]):
            y = mb.scaled_mm(a, w, sa, sb, bias=bias, out_dtype=torch.float32, _plan=plan)
            check_product(y, a, w, sa, sb, bias)
            assert torch.equal(y, mb.scaled_mm(a, w, sa, sb, bias=bias, out_dtype=torch.float32))


@pytest.mark.parametrize("plan", PLANS)
def test_every_tile_and_split_by_group(plan):
    g = gen(42)
    K = 1040
    for counts, extra, N in (([3, 0, 17, 130, 1, 0, 40], 5, 390), ([2, 1] * 30, 0, 1040), ([0, 600, 1, 300], 77, 515)):
        M, E = sum(counts) + extra, len(counts)
        a, sa, sb, off = ints((M, K), g), scales((M,), g), scales((E, N), g), offsets_of(counts)
        w = ints((E, N, K), g).transpose(1, 2)
        for out_dtype in (torch.bfloat16, torch.float32):
            y = mb.grouped_scaled_mm(a, w, sa, sb, off, out_dtype=out_dtype, _plan=plan,
                                     out=torch.full((M, N), float("nan"), dtype=out_dtype, device=DEV))
            check_grouped(y, a, w, sa, sb, off)


def test_forced_plans_that_do_not_exist_are_refused():
    g = gen(43)
    a, w, sa, sb = ints((64, 256), g), ints((128, 256), g).t(), scales((64,), g), scales((128,), g)
    for plan in ((48, 0, 0, 0), (512, 0, 0, 1), (16, 0, -1, 0), (0, 3, 0, 0), (0, 4, 0, 0), (256, 2, 0, 0)):
        with pytest.raises(ValueError):
            mb.scaled_mm(a, w, sa, sb, _plan=plan)


# ------------------------------------------------------------------------------ refusals
def test_refusals():
    z = lambda *s, dt=torch.int8: torch.zeros(*s, dtype=dt, device=DEV)  # noqa: E731
    f = lambda *s: torch.ones(*s, device=DEV)  # noqa: E731
    a, b, sa, sb = z(4, 16), z(16, 8), f(4), f(8)
    with pytest.raises(AssertionError):
        mb.quantize(torch.zeros(2, 2))
    for dt in (torch.float64, torch.int8, torch.complex64):
        with pytest.raises(NotImplementedError):
            mb.quantize(z(2, 2, dt=dt))
    with pytest.raises(AssertionError):
        mb.scaled_mm(a, z(15, 8), sa, sb)
    with pytest.raises(AssertionError):
        mb.scaled_mm(a, b, f(5), sb)
    with pytest.raises(AssertionError):
        mb.scaled_mm(a, b, sa, f(4, 8))
    with pytest.raises(AssertionError):
        mb.scaled_mm(a, b, sa.cpu(), sb)
    with pytest.raises(AssertionError):
        mb.scaled_mm(a, b.cpu(), sa, sb)
    with pytest.raises(NotImplementedError):
        mb.scaled_mm(a, b, sa.half(), sb)
    with pytest.raises(NotImplementedError):
        mb.scaled_mm(z(4, 16, dt=torch.uint8), b, sa, sb)
    with pytest.raises(NotImplementedError):
        mb.scaled_mm(a, b, sa, sb, out_dtype=torch.int32)
    with pytest.raises(NotImplementedError):
        mb.scaled_mm(a, b, sa, sb, bias=torch.ones(8, dtype=torch.float16, device=DEV))
    with pytest.raises(AssertionError):
        mb.scaled_mm(a, b, sa, sb, bias=f(7))
    with pytest.raises(AssertionError):
        mb.scaled_mm(a, b, sa, sb, out=f(4, 7))
    with pytest.raises(ValueError):
        mb.scaled_mm(a, b, sa, sb, out=f(4, 8), out_dtype=torch.float16)
    with pytest.raises(ValueError):
        mb.scaled_mm(z(1, 131072), z(131072, 1), f(1), f(1))
    off = torch.tensor([0, 2, 4], dtype=torch.int32, device=DEV)
    b3, sb3 = z(2, 16, 8), f(2, 8)
    with pytest.raises(NotImplementedError):
        mb.grouped_scaled_mm(a, b3, sa, sb3, off.long())
    with pytest.raises(AssertionError):
        mb.grouped_scaled_mm(a, b3, sa, sb3, off[:2])
    with pytest.raises(AssertionError):
        mb.grouped_scaled_mm(a, b3, sa, f(3, 8), off)
    with pytest.raises(ValueError):
        mb.grouped_scaled_mm(a, z(1025, 16, 1), sa, f(1025, 1), torch.zeros(1026, dtype=torch.int32, device=DEV))
