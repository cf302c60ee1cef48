"""Rows, linears, grouped products and routed layers in int8 (ops.quantize_int8, linear_int8, rms_norm, grouped_mm, moe_experts_stacked) against their definitions in
64 bits.

Tolerances are bounds by arithmetic.  Sums of int8 products are exact; what follows is the conversion to float32, two products and a bias, each off by 2^-24 relative at
most, and the result's rounding by half a step, finfo(t).eps / 2 relative (and half the smallest subnormal).  Rounded rows are equal to the definition's."""
import ctypes
import math

import pytest
import torch

from htr_amd import _native, ops

BF16, F16, F32, I8, E4M3 = torch.bfloat16, torch.float16, torch.float32, torch.int8, torch.float8_e4m3fn


@pytest.fixture
def gen():
    return torch.Generator(device="cuda").manual_seed(20261208)


def randn(gen, *shape, dtype=F32, scale=1.0):
    return (torch.randn(*shape, device=gen.device, generator=gen) * scale).to(dtype)


def half_step(y, dtype):
    f = torch.finfo(dtype)
    return y.abs() * (f.eps / 2) + f.smallest_normal * f.eps / 2


def rounded(x):
    """(integers, scales) of float64 rows, both float64."""
    amax = x.abs().amax(-1)                                                     # NaN where there is one
    s = (amax.clamp(min=2.0 ** -100) / 127).float().double()
    s = torch.where(s.isfinite(), s, torch.nan)
    z = x / s[..., None]
    return torch.where(z.isfinite(), torch.trunc(z + torch.copysign(torch.full_like(z, 0.5), z)), 0.0), s


def value(q, s):
    return q.double() * s.double()[..., None]


def assert_within(got, want, bound):
    got = got.double()
    assert got.shape == want.shape
    assert torch.equal(got.isnan(), want.isnan())
    off = ((got - want).abs() - bound).nan_to_num(0.0)
    assert off.max().item() <= 0 if off.numel() else True, f"{off.max().item()} beyond the bound at {off.argmax().item()}"


def product(x, w):
    """Of int8 pairs: the integers' sums are exact in 64 bits (a sum of products of scaled values is not, where it comes to zero)."""
    return (x[0].double() @ w[0].double().T) * x[1].double()[..., None] * w[1].double()


def product_bound(x, w, dtype, bias=None):
    """(y, bound) of int8 pairs' product."""
    y = product(x, w)
    bound = y.abs() * 3.01 * 2.0 ** -24
    if bias is not None:
        y = y + bias.double()
        bound = bound + y.abs() * 2.0 ** -24
    return y, bound * 1.01 + half_step(y.abs() + bound, dtype)


def weight(gen, *shape):
    return ops.quantize_weight_int8(randn(gen, *shape, scale=shape[-1] ** -0.5) * torch.exp(randn(gen, *shape[:-1], 1)))


def equal_rows(got, want):
    assert got[0].dtype == I8 and got[1].dtype == F32 and got[0].shape == want[0].shape and got[1].shape == want[1].shape
    assert torch.equal(got[1].double().nan_to_num(-1.0), want[1].nan_to_num(-1.0))
    assert torch.equal(got[0].double(), want[0])


# ---- rows
def special_rows(dtype, n):
    """Zeros, infinities, NaN, halves, the ends of the type's range."""
    f = torch.finfo(dtype)
    x = torch.zeros(14, n, dtype=dtype)
    x[1, 3], x[2, n - 1], x[3, 0] = math.inf, math.nan, -math.inf
    halves = torch.arange(n) % 254 - 126.5
    x[4] = halves.to(dtype)                                    # scale 126.5 / 127, in short rows less
    x[5] = halves.to(dtype)
    x[5, 0] = -127                                             # scale 1: every other value is a half
    x[6] = (1.5 * (torch.arange(n) % 84 * 2 - 83)).to(dtype)
    x[6, 1] = 381                                              # scale 3: halves again, 1 / 3 is none of the type's (381 is 382 in bfloat16)
    x[7] = (0.875 * halves).to(dtype)
    x[7, 5] = 0.875 * 127
    x[8], x[9] = f.max, f.tiny
    x[9, 2] = -f.tiny * f.eps                                  # the smallest subnormal
    x[10, 5] = f.tiny * f.eps
    x[11, ::2] = f.max
    x[12], x[12, 1] = -1, 127
    x[13, 7] = -0.0
    return x


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("n", [16, 48, 640, 1408, 4096, 8192, 8208, 16384, 16400, 32768, 32784, 40960])
def test_rows_to_int8(gen, dtype, n):
    x = torch.cat((randn(gen, 9, n, dtype=dtype) * torch.exp(3 * randn(gen, 9, 1)).to(dtype), special_rows(dtype, n).cuda()))
    equal_rows(ops.quantize_int8(x), rounded(x.double()))
    equal_rows(ops.quantize_int8(x[4]), rounded(x[4].double()))


@pytest.mark.gpu
def test_rows_to_int8_from_any_strides(gen):
    big = randn(gen, 6, 5, 300, dtype=BF16)
    for x in (big[:, 1, 5:261], big[::2, :, 9:265], big.transpose(0, 1)[..., :48], big[:, :, ::2][..., :144], big[0, 0, 1:17].expand(4, 16)):
        equal_rows(ops.quantize_int8(x), rounded(x.double()))
    q, s = ops.quantize_int8(big[:0, :, :32])
    assert q.shape == (0, 5, 32) and s.shape == (0, 5)


def test_weights_to_int8():
    w = torch.randn(3, 20, 64, generator=torch.Generator().manual_seed(1))
    w[1, 3, 7], w[2, 4, 1], w[0, 5] = math.inf, math.nan, 0
    q, s = ops.quantize_weight_int8(w)
    equal_rows((q, s), rounded(w.double()))
    assert s[1, 3].isnan() and s[2, 4].isnan() and (q[0, 5] == 0).all() and s.isnan().sum() == 2
    w = w.nan_to_num(0.0, 0.0)
    q, s = ops.quantize_weight_int8(w.half())
    equal_rows((q, s), rounded(w.half().double()))
    # half a step of the scale, whose own rounding moves a value of 127 steps by 127 2^-24 of one
    assert ((ops.dequantize_int8(q, s) - w.half().float()).abs() <= s[..., None] * (0.5 + 127 * 2.0 ** -22)).all()


# ---- norm
def norm64(x, w, eps, residual):
    t = x if residual is None else (x.float() + residual.float()).to(x.dtype)
    d = t.double()
    return d / torch.sqrt((d * d).mean(-1, keepdim=True) + eps) * w.double(), t


def equal_but_for_halves(got, y):
    """As equal_rows, except where 64 bits themselves do not say on which side of a half a quotient lies, or a scale of its rounding: 2^-40 for some thousand roundings of
    2^-53."""
    want, s = rounded(y)
    assert got[0].dtype == I8 and got[1].dtype == F32
    q, scale = got[0].double(), got[1].double()
    assert torch.equal(scale.isnan(), s.isnan())
    same = (scale == s) | s.isnan()
    exact = (y.abs().amax(-1).clamp(min=2.0 ** -100) / 127)
    near = (torch.nextafter(s.float(), torch.full_like(s.float(), math.inf)).double() + s) / 2, (torch.nextafter(s.float(), torch.zeros_like(s.float())).double() + s) / 2
    assert (same | ((exact / near[0] - 1).abs() < 2.0 ** -40) | ((exact / near[1] - 1).abs() < 2.0 ** -40)).all()
    want, _ = (torch.where(same[..., None], want, q), 0)
    z = (y / s[..., None]).abs().nan_to_num(0.0)
    unclear = ((z - torch.floor(z)) - 0.5).abs() < 2.0 ** -33
    assert (unclear | (q == want)).all() and ((q - want).abs() <= 1).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("rows,n", [(1, 16), (1, 4096), (7, 400), (33, 1408), (3, 8192), (2, 8208), (5, 16384), (2, 16400), (2, 32768), (2, 40960), (2100, 528)])
@pytest.mark.parametrize("residual", [False, True])
def test_norm_to_int8(gen, dtype, rows, n, residual):
    x, w = randn(gen, rows, n, dtype=dtype), randn(gen, n, dtype=dtype)
    r = randn(gen, rows, n, dtype=dtype, scale=3) if residual else None
    out = ops.rms_norm(x, w, 1e-6, residual=r, quantize=I8)
    want, t = norm64(x, w, 1e-6, r)
    if residual:
        out, total = out
        assert torch.equal(total, t)
    equal_but_for_halves(out, want)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [256, 40960])
@pytest.mark.parametrize("dtype,size,factor", [(F32, 1e38, 1.0), (F32, 1e-39, 1.0), (F32, 1e30, 1e20), (F32, 1.0, 1e38), (BF16, 2.0 ** 125, 1.0), (BF16, 2.0 ** 124, 2.0 ** 20),
                                               (BF16, 2.0 ** -100, 2.0 ** -40), (F16, 2.0 ** -12, 2.0 ** -12), (BF16, 1.0, 2.0 ** 127), (BF16, 1.0, 2.0 ** 126)])
def test_norm_to_int8_of_rows_of_any_size(gen, dtype, n, size, factor):
    sign = lambda: torch.randint(0, 2, (3, n), device="cuda", generator=gen) * 2 - 1
    x = (sign() * size * (1 + torch.rand(3, n, device="cuda", generator=gen))).to(dtype)
    w = (factor * (1 + torch.rand(n, device="cuda", generator=gen))).to(dtype)
    assert x.isfinite().all() and (w.isfinite().all() or factor == 2.0 ** 127)          # 2^128 is an infinity: the row's scale is NaN
    equal_but_for_halves(ops.rms_norm(x, w, 0.0, quantize=I8), norm64(x, w, 0.0, None)[0])


@pytest.mark.gpu
def test_norm_to_int8_of_zeros_infinities_and_nan(gen):
    x = randn(gen, 5, 256, dtype=BF16)
    x[0], x[1, 3], x[2, 200] = 0, math.inf, math.nan
    w = torch.ones(256, dtype=BF16, device="cuda")
    q, s = ops.rms_norm(x, w, quantize=I8)
    assert (q[:3] == 0).all() and s[1:3].isnan().all() and s[0] == torch.tensor(2.0 ** -100 / 127).float()
    equal_but_for_halves((q[3:], s[3:]), norm64(x[3:], w, 1e-6, None)[0])
    q, s = ops.rms_norm(x, w, 0.0, quantize=I8)          # 0 / 0
    assert s[0].isnan() and (q[0] == 0).all()
    w[9] = math.nan
    q, s = ops.rms_norm(x, w, quantize=I8)
    assert s.isnan().all() and (q == 0).all()


@pytest.mark.gpu
def test_norm_to_int8_takes_strides_and_any_alignment(gen):
    big, w = randn(gen, 6, 3, 400, dtype=BF16), randn(gen, 257, dtype=BF16)
    for x in (big[:, 1, 5:261], big[::2, :, 8:264], big[:, :, 0:256].transpose(0, 1), big.transpose(1, 2)[:, :256, :2].transpose(1, 2)):
        for factor in (w[:256], w[1:]):
            r = randn(gen, *x.shape, dtype=BF16)
            (q, s), t = ops.rms_norm(x, factor, residual=r, quantize=I8)
            (q2, s2), t2 = ops.rms_norm(x.contiguous(), factor.clone(), residual=r, quantize=I8)
            assert torch.equal(q, q2) and torch.equal(s, s2) and torch.equal(t, t2)
    (q, s), t = ops.rms_norm(big[:0, :, :32], w[:32], residual=big[:0, :, :32], quantize=I8)
    assert q.shape == t.shape == (0, 3, 32) and s.shape == (0, 3)
    for a, b in zip(ops.rms_norm(big[..., :256], w[:256], quantize=E4M3), ops.rms_norm(big[..., :256], w[:256], quantize=True)):
        assert torch.equal(a.float(), b.float())


@pytest.mark.gpu
def test_more_rows_than_a_launch_takes(gen):
    rows = (1 << 21) + 3
    x, w = randn(gen, rows, 128, dtype=BF16), randn(gen, 128, dtype=BF16)
    for a, b in zip(ops.rms_norm(x, w, quantize=I8), ops.rms_norm(x[rows - 7:].clone(), w, quantize=I8)):
        assert torch.equal(a[rows - 7:], b)
    for a, b in zip(ops.quantize_int8(x), ops.quantize_int8(x[rows - 7:].clone())):
        assert torch.equal(a[rows - 7:], b)


# ---- products
@pytest.mark.gpu
@pytest.mark.parametrize("m,n", [(1, 16), (100, 256), (128, 656), (384, 4096), (1030, 1168)])
@pytest.mark.parametrize("rows", [1, 2, 3, 4, 5, 7, 8, 9, 16, 17, 32, 33, 64, 65, 100, 193, 300])
def test_linear_int8(gen, m, n, rows):
    w, ws = weight(gen, m, n)
    for dtype, bias in ((BF16, False), (F16, True), (F32, True)):
        x = randn(gen, rows, n, dtype=dtype)
        b = randn(gen, m, dtype=dtype) if bias else None
        pair = ops.quantize_int8(x)
        want, bound = product_bound(pair, (w, ws), dtype, b)
        y = ops.linear_int8(x, w, ws, b)
        assert y.dtype == dtype
        assert_within(y, want, bound)
        assert torch.equal(ops.linear_int8(pair, w, ws, b, out_dtype=dtype), y)        # rounded ahead or on the way
    assert ops.linear_int8(pair, w, ws).dtype == BF16 and ops.linear_int8(pair, w, ws, b.half()).dtype == F16


@pytest.mark.gpu
@pytest.mark.parametrize("m,n", [(5, 32), (7, 2048), (2047, 2064), (2600, 272), (70000, 48), (300, 20480), (9, 131056)])
@pytest.mark.parametrize("rows", [1, 2, 3, 4, 6, 8, 11, 16, 23, 32])
def test_few_rows(gen, m, n, rows):
    """Rows that lie in LDS: matrices of more and of fewer tiles than workgroups, more than 32 tiles to one, rows of less than a step, and sizes that LDS does not hold."""
    w, ws = weight(gen, m, n)
    x, b = randn(gen, rows, n), randn(gen, m)
    pair = ops.quantize_int8(x)
    want, bound = product_bound(pair, (w, ws), F32, b)
    y = ops.linear_int8(x, w, ws, b)
    assert_within(y, want, bound)
    assert torch.equal(ops.linear_int8(pair, w, ws, b), y)
    around = torch.full((rows + 2, m), 7.0, device="cuda")            # what lies around the result is left
    L, p = _native.lib(), lambda t: t.data_ptr()
    if (m * 4) % 16 == 0:
        y = around[1:rows + 1]
        assert L.htr_product(p(pair[0]), 4, p(pair[1]), p(w), p(ws), p(b), None, p(y), rows, m, n, 1, 4, 2, torch.cuda.current_stream().cuda_stream) == 0
        assert_within(y, want, bound)
        assert (around[0] == 7).all() and (around[-1] == 7).all()


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 3, 40, 300])
@pytest.mark.parametrize("n", [16, 4096, 131056])
def test_the_largest_sums(rows, n):
    """-128 by -128 throughout: 2^14 n, which 32 bits just hold."""
    w, ws = torch.full((130, n), -128, dtype=I8, device="cuda"), torch.full((130,), 0.5, device="cuda")
    w[77] = 127
    x = torch.full((rows, n), -128, dtype=I8, device="cuda"), torch.full((rows,), 2.0, device="cuda")
    want = torch.full((rows, 130), float(n) * 16384, dtype=torch.float64, device="cuda")
    want[:, 77] = -128.0 * 127 * n
    assert_within(ops.linear_int8(x, w, ws, out_dtype=F32), want, want.abs() * 2.0 ** -24)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [3, 18, 90, 260])
def test_a_row_with_nan_keeps_to_itself(gen, rows):
    w, ws = weight(gen, 144, 512)
    x = randn(gen, rows, 512, dtype=BF16)
    clean = ops.linear_int8(x, w, ws)
    x[1, 5], x[2, 300] = math.nan, -math.inf
    ws[7] = math.nan
    y = ops.linear_int8(x, w, ws)
    assert y[1:3].isnan().all() and y[:, 7].isnan().all()
    y[:, 7] = clean[:, 7]
    assert torch.equal(y[0], clean[0]) and torch.equal(y[3:], clean[3:])


@pytest.mark.gpu
def test_linear_int8_takes_any_leading_dimensions_and_scales(gen):
    w, ws = weight(gen, 96, 256)
    x = randn(gen, 2, 5, 300, dtype=BF16)[..., 3:259]
    y = ops.linear_int8(x, w, ws)
    assert y.shape == (2, 5, 96)
    assert torch.equal(y.reshape(10, 96), ops.linear_int8(x.reshape(10, 256).contiguous(), w, ws))
    assert ops.linear_int8(x[:, :0], w, ws).shape == (2, 0, 96)
    assert torch.equal(ops.linear_int8(x[0, 0], w, ws), y[0, 0])
    q, s = ops.quantize_int8(x)
    assert torch.equal(ops.linear_int8((q.transpose(0, 1), s.transpose(0, 1)), w, ws, out_dtype=BF16), y.transpose(0, 1))
    scales = torch.stack((ws, ws), 1)[:, 0]                                         # every other element: weights lie in consecutive memory
    with pytest.raises(RuntimeError, match="contiguous"):
        ops.linear_int8(x, w, scales)
    for size in (2.0 ** -120, 2.0 ** 100, 0.0, -1.0):                               # scales from elsewhere
        want, bound = product_bound((q, s * size), (w, ws), F32)
        assert_within(ops.linear_int8((q, s * size), w, ws, out_dtype=F32), want, bound + 2.0 ** -149 * (1 + ws.double() * 2))


@pytest.mark.gpu
def test_products_of_many_kinds_of_tiles(gen):
    """Every kernel that the sizes choose between, rows and matrix ending inside a tile."""
    seen = set()
    for rows, m, n in [(1, 5000, 512), (12, 9000, 256), (16, 16400, 128), (20, 700, 2064), (30, 2050, 400), (31, 10000, 272), (32, 20011, 256), (60, 500, 4096), (90, 3001, 1040),
                       (130, 4100, 320), (200, 1024, 4096), (257, 6100, 192), (300, 9001, 272), (700, 4099, 528), (1100, 5003, 640), (2100, 4096, 400), (4111, 9003, 304),
                       (520, 28672, 256)]:
        plan = (ctypes.c_int * 6)()
        assert _native.lib().htr_product_plan(rows, m, n, 1, 0, 0, _native.I8, _native.I8, plan) == 0
        seen.add(tuple(plan[:4]))
        w, x = weight(gen, m, n), ops.quantize_int8(randn(gen, rows, n))
        want, bound = product_bound(x, w, BF16)
        assert_within(ops.linear_int8(x, *w), want, bound)
    assert len(seen) >= 8, seen


@pytest.mark.gpu
@pytest.mark.parametrize("n", [16, 48, 128, 144, 256, 272, 384, 400, 512, 528])
@pytest.mark.parametrize("rows,m", [(5000, 6000), (1100, 9000), (400, 20000), (200, 9000)])
def test_short_rows_of_many_tiles(gen, n, rows, m):
    """Several tiles to a workgroup, each with fewer slabs than the ring has stages, as many, and more: a tile's scales may not reach the one before."""
    w, x = weight(gen, m, n), ops.quantize_int8(randn(gen, rows, n) * torch.exp(randn(gen, rows, 1)))
    want, bound = product_bound(x, w, F32)
    for _ in range(3):
        assert_within(ops.linear_int8(x, *w, out_dtype=F32), want, bound)


def _ends(counts):
    return torch.tensor(counts, dtype=torch.int32).cumsum(0).to(torch.int32).cuda()


COUNTS = [[1], [0, 1, 0], [5, 0, 0, 11, 1], [16, 17, 0, 33, 1, 64], [0, 0, 0], [200, 0, 1, 130, 129], [300, 5], [3] * 70, [0] * 64 + [7, 0, 40]]


def check_grouped(x, w, counts, dtype, y):
    first = 0
    for e, c in enumerate(counts):
        rows = slice(first, first + c)
        assert_within(y[rows], *product_bound((x[0][rows], x[1][rows]), (w[0][e], w[1][e]), dtype))
        first += c
    assert (y[first:] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("counts", COUNTS, ids=lambda c: f"{len(c)}x{sum(c)}")
@pytest.mark.parametrize("m,n", [(200, 256), (24, 1168), (130, 16)])
@pytest.mark.parametrize("behind", [0, 19])
def test_grouped_mm(gen, counts, m, n, behind):
    R, E = sum(counts) + behind, len(counts)
    floats, w = randn(gen, R, n, dtype=F16), weight(gen, E, m, n)
    x = ops.quantize_int8(floats)
    y = ops.grouped_mm(x, w, _ends(counts))
    assert y.dtype == BF16 and y.shape == (R, m)
    check_grouped(x, w, counts, BF16, y)
    check_grouped(x, w, counts, F16, ops.grouped_mm(floats, w, _ends(counts)))
    check_grouped(x, w, counts, F32, ops.grouped_mm(x, w, _ends(counts), out_dtype=F32))


@pytest.mark.gpu
@pytest.mark.parametrize("counts", [[0, 3, 0, 0, 17, 1, 0, 5], [1] * 300, [40] + [0] * 9, [2, 0] * 100 + [33], [8] * 12, [7, 7, 7, 7, 20, 0, 1]], ids=lambda c: f"{len(c)}x{sum(c)}")
@pytest.mark.parametrize("m,n", [(7, 16), (66, 784), (520, 2048), (300, 2064), (1030, 4112), (40, 16400)])
@pytest.mark.parametrize("behind", [0, 3, 40])
def test_grouped_mm_of_few_rows(gen, counts, m, n, behind):
    """Several experts, and several tiles of one, to a workgroup; experts of more rows than go together; rows that LDS does not hold."""
    R = sum(counts) + behind
    x, w = ops.quantize_int8(randn(gen, R, n)), weight(gen, len(counts), m, n)
    check_grouped(x, w, counts, BF16, ops.grouped_mm(x, w, _ends(counts)))
    x[1][:] = 1.0
    x[1][R // 2] = math.nan                            # a row without a value keeps to itself, and so does a matrix that no row asks for
    w[1][counts.index(0) if 0 in counts else 0] = math.nan
    check_grouped(x, w, counts, F32, ops.grouped_mm(x, w, _ends(counts), out_dtype=F32))


@pytest.mark.gpu
@pytest.mark.parametrize("counts,m", [([e * 7 % 37 for e in range(130)], 512), ([2000, 0, 3100], 4096), ([0] * 63 + [1900, 0, 2500] + [1] * 70, 1000),
                                      ([300 - 4 * e for e in range(75)], 1024), ([0] * 64 + [700], 2900)], ids=lambda c: str(len(c) if isinstance(c, list) else c))
def test_grouped_mm_of_more_tiles_than_run_at_once(gen, counts, m):
    n, R = 272, sum(counts) + 45
    x, w = ops.quantize_int8(randn(gen, R, n)), weight(gen, len(counts), m, n)
    check_grouped(x, w, counts, BF16, ops.grouped_mm(x, w, _ends(counts)))


@pytest.mark.gpu
@pytest.mark.parametrize("E", [15000, 28000, 40000])
@pytest.mark.parametrize("rows_of", [lambda e: e % 3 == 0, lambda e: e * 0 + 1, lambda e: e % 5], ids=["a third", "one", "up to four"])
def test_grouped_mm_of_tens_of_thousands_of_experts(gen, E, rows_of):
    """Up to some sixty experts to a workgroup, and more than it takes."""
    m, n = 20, 48
    counts = rows_of(torch.arange(E, device="cuda")).int()
    of, R = torch.repeat_interleave(torch.arange(E, device="cuda"), counts), int(counts.sum()) + 7
    x, w = ops.quantize_int8(randn(gen, R, n)), weight(gen, E, m, n)
    y = ops.grouped_mm(x, w, counts.cumsum(0).int(), out_dtype=F32)
    R -= 7
    want = (x[0][:R, None].double() * w[0][of].double()).sum(-1) * x[1][:R, None].double() * w[1][of].double()
    assert_within(y[:R], want, want.abs() * 3.01 * 2.0 ** -24 * 1.01 + half_step(want, F32))
    assert (y[R:] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("ends,meant", [([4, 2, 9], [4, 4, 9]), ([-5, 3, 100], [0, 3, 40]), ([2 ** 31 - 1, 0, 7], [40, 40, 40]), ([-1, -2, -3], [0, 0, 0])])
def test_ends_out_of_order_or_range(gen, ends, meant):
    x, w = ops.quantize_int8(randn(gen, 40, 64)), weight(gen, 3, 40, 64)
    to = lambda e: torch.tensor(e, dtype=torch.int32, device="cuda")
    assert torch.equal(ops.grouped_mm(x, w, to(ends)), ops.grouped_mm(x, w, to(meant)))


# ---- routed layers
def moe64(x, ids, wt, gate_up, down, dtype):
    """(y, bound) of the layer.  Sums are exact, so gate and up are off by three roundings of float32; the rest of silu(gate) up by 2^-20 (1 + |gate|) relative: the
    exponential's argument in units of log2 is off by 2^-23 |gate| and its result by 2^-22, two quotients and products by 2^-22.  Hidden values within that of a half may
    be one step off, and the row's scale moves with its largest value."""
    T, H = x.shape
    q = rounded(x.double())
    y, bound = torch.zeros(T, H, dtype=torch.float64, device=x.device), torch.zeros(T, H, dtype=torch.float64, device=x.device)
    for t in range(T):
        for j in range(ids.shape[1]):
            e = int(ids[t, j])
            if not 0 <= e < gate_up[0].shape[0]:
                y[t] = math.nan
                continue
            g, u = product((q[0][t:t + 1], q[1][t:t + 1]), (gate_up[0][e], gate_up[1][e]))[0].chunk(2)
            h = g * torch.sigmoid(g) * u
            off = h.abs() * 2.0 ** -20 * (1 + g.abs())
            hq, s = rounded(h)
            z = (h / s).abs()
            dz = off / s + z * (off.max() / h.abs().max().clamp(min=2.0 ** -100) + 2.0 ** -23)
            flips = (((z - torch.floor(z)) - 0.5).abs() <= dz).double()
            wd = value(down[0][e], down[1][e])
            out = product((hq[None], s[None]), (down[0][e], down[1][e]))[0]
            p = float(wt[t, j])
            y[t] += p * out
            moved = off.max() / h.abs().max().clamp(min=2.0 ** -100) + 2.0 ** -23
            bound[t] += abs(p) * (wd.abs() @ flips * s + (wd.abs() @ (hq * s).abs()) * moved + out.abs() * 2.0 ** -22) * (1 + 2.0 ** -22) + (p * out).abs() * 2.0 ** -23
    bound += (bound + y.abs()).nan_to_num(0.0) * ids.shape[1] * 2.0 ** -23
    return y, bound * 1.01 + half_step(y.abs() + bound, dtype)


def experts(gen, E, H, F):
    return weight(gen, E, 2 * F, H), weight(gen, E, H, F)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("T,E,top,H,F", [(1, 4, 2, 256, 128), (5, 8, 3, 144, 400), (40, 3, 1, 256, 256), (9, 70, 8, 128, 128), (70, 2, 2, 400, 144), (60, 70, 7, 256, 16), (300, 4, 2, 32, 80), (9, 12, 5, 2064, 48), (50, 40, 6, 80, 2080)])
@pytest.mark.parametrize("ids64", [True, False])
def test_moe_experts_stacked(gen, dtype, T, E, top, H, F, ids64):
    x, wt = randn(gen, T, H, dtype=dtype), torch.rand(T, top, device="cuda", generator=gen)
    ids = torch.argsort(torch.rand(T, E, device="cuda", generator=gen))[:, :top]
    gate_up, down = experts(gen, E, H, F)
    y = ops.moe_experts_stacked(x, ids if ids64 else ids.int(), wt, gate_up, down)
    assert y.dtype == dtype
    assert_within(y, *moe64(x, ids, wt, gate_up, down, dtype))


@pytest.mark.gpu
def test_moe_with_one_expert_twice_and_experts_out_of_range(gen):
    T, E, H, F = 6, 4, 256, 128
    x, wt = randn(gen, T, H, dtype=BF16), torch.rand(T, 3, device="cuda", generator=gen)
    ids = torch.randint(0, E, (T, 3), device="cuda", generator=gen)
    ids[0] = 2
    ids[1, 1], ids[2, 0], ids[3, 2] = -1, E, 2 ** 40
    gate_up, down = experts(gen, E, H, F)
    want, bound = moe64(x, ids, wt, gate_up, down, BF16)
    y = ops.moe_experts_stacked(x, ids, wt, gate_up, down)
    assert y[1:4].isnan().all()
    assert_within(y, want, bound)
    assert ops.moe_experts_stacked(x, torch.full_like(ids, -1), wt, gate_up, down).isnan().all()
    assert ops.moe_experts_stacked(x[:0], ids[:0], wt[:0], gate_up, down).shape == (0, H)
    assert (ops.moe_experts_stacked(x, ids[:, :0], wt[:, :0], gate_up, down) == 0).all()
    ids = ids.clamp(0, E - 1)
    clean = ops.moe_experts_stacked(x, ids, wt, gate_up, down)
    x[4, 9] = math.nan
    y = ops.moe_experts_stacked(x, ids, wt, gate_up, down)
    assert y[4].isnan().all()
    keep = torch.arange(T, device="cuda") != 4
    assert torch.equal(y[keep], clean[keep])


# ---- as they are used
def _block(gen, H=256, F=144, E=6):
    """A decoder block's tail: norm, an int8 linear, norm, router, routed experts."""
    wt = dict(n1=randn(gen, H, dtype=BF16), o=weight(gen, H, H), n2=randn(gen, H, dtype=BF16), router=randn(gen, E, H, scale=H ** -0.5), experts=experts(gen, E, H, F))

    def run(x, h):
        xq, h = ops.rms_norm(x, wt["n1"], residual=h, quantize=I8)
        y = ops.linear_int8(xq, *wt["o"])
        y, h = ops.rms_norm(y, wt["n2"], residual=h)
        ids, p = ops.route_experts(y.float() @ wt["router"].T, 2)
        return ops.moe_experts_stacked(y, ids, p, *wt["experts"]), h
    return run


@pytest.mark.gpu
def test_a_block_of_them_eager_on_streams_captured_and_compiled(gen):
    run = _block(gen)
    inputs = [(randn(gen, 9, 256, dtype=BF16), randn(gen, 9, 256, dtype=BF16)) for _ in range(4)]
    want = [run(*i) for i in inputs]
    side = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for k, i in enumerate(inputs):                      # two streams at once
        side[k % 2].wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side[k % 2]):
            got.append(run(*i))
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    x, h = (t.clone() for t in inputs[0])
    with torch.cuda.stream(side[0]):
        run(x, h)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run(x, h)
    for k in (1, 2, 3, 0, 2):
        x.copy_(inputs[k][0])
        h.copy_(inputs[k][1])
        graph.replay()
        run(*inputs[(k + 1) % 4])                       # eager work between the replays
        torch.cuda.synchronize()
        assert torch.equal(out[0], want[k][0]) and torch.equal(out[1], want[k][1])
    for a, b in zip(torch.compile(run, backend="eager")(*inputs[1]), want[1]):
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_layers_of_many_rows_on_streams_and_captured(gen):
    """Tiles that go on from one to the next, on two streams at once and replayed."""
    w, experts = weight(gen, 6000, 512), (weight(gen, 4, 1024, 512), weight(gen, 4, 512, 512))
    ids, wt = torch.randint(0, 4, (1500, 2), device="cuda", generator=gen), torch.rand(1500, 2, device="cuda", generator=gen)

    def run(x):
        y = ops.moe_experts_stacked(x, ids, wt, *experts)
        return ops.linear_int8(y, *w)

    inputs = [randn(gen, 1500, 512, dtype=BF16) for _ in range(4)]
    want = [run(x) for x in inputs]
    side = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for k, x in enumerate(inputs):
        side[k % 2].wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side[k % 2]):
            got.append(run(x))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    x = inputs[0].clone()
    with torch.cuda.stream(side[0]):
        run(x)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run(x)
    for k in (1, 2, 3, 0, 2):
        x.copy_(inputs[k])
        graph.replay()
        run(inputs[(k + 1) % 4])                        # eager work between the replays
        torch.cuda.synchronize()
        assert torch.equal(out, want[k])


@pytest.mark.gpu
def test_beyond_32_bits(gen):
    """Matrices, rows and results whose places in memory pass 2^32 bytes."""
    E, m, n = 40, 8192, 16384
    w, ws = torch.zeros(E, m, n, dtype=I8, device="cuda"), torch.zeros(E, m, device="cuda")              # 5.4 GB
    q, s = weight(gen, 256, n)
    w[E - 1, m - 256:], ws[E - 1, m - 256:] = q, s
    ends = torch.zeros(E, dtype=torch.int32, device="cuda")
    for rows in (3, 200):
        ends[E - 1] = rows
        x = ops.quantize_int8(randn(gen, rows, n))
        y = ops.grouped_mm(x, (w, ws), ends)
        assert_within(y[:, m - 256:], *product_bound(x, (q, s), BF16))
        assert (y[:, :m - 256] == 0).all()
    del w, ws
    rows, n = 1_200_000, 128
    x, pair = randn(gen, rows, n, dtype=BF16), weight(gen, 2048, n)
    y = ops.linear_int8(x, *pair)                                                      # 4.9 GB
    last = slice(rows - 5, rows)
    assert torch.equal(y[last], ops.linear_int8(x[last].clone(), *pair))
    for a, b in zip(ops.quantize_int8(y), ops.quantize_int8(y[last].clone())):
        assert torch.equal(a[last], b)
    one = torch.ones(2048, dtype=BF16, device="cuda")
    for a, b in zip(ops.rms_norm(y, one, quantize=I8), ops.rms_norm(y[last].clone(), one, quantize=I8)):
        assert torch.equal(a[last], b)


# ---- refusals
def wrong_calls(device):
    x, w = torch.zeros(2, 128, dtype=BF16, device=device), torch.zeros(128, dtype=BF16, device=device)
    q, s = torch.zeros(64, 128, dtype=I8, device=device), torch.zeros(64, device=device)
    q8, s8 = torch.zeros(64, 128, device=device).to(E4M3), torch.zeros(1, 1, device=device)
    rows, ends = (torch.zeros(2, 128, dtype=I8, device=device), torch.zeros(2, device=device)), torch.zeros(1, dtype=torch.int32, device=device)
    ids, p = torch.zeros(2, 1, dtype=torch.int64, device=device), torch.zeros(2, 1, device=device)
    gu, dn = (torch.zeros(1, 32, 128, dtype=I8, device=device), torch.zeros(1, 32, device=device)), (torch.zeros(1, 128, 16, dtype=I8, device=device), torch.zeros(1, 128, device=device))
    moe = ops.moe_experts_stacked
    return [lambda: ops.rms_norm(x[:, :24], w[:24], quantize=I8), lambda: ops.rms_norm(x, w, quantize=BF16), lambda: ops.rms_norm(x, w, quantize=torch.uint8),
            lambda: ops.quantize_int8(x[:, :24]), lambda: ops.quantize_int8(x.double()), lambda: ops.quantize_int8(x[0, 0]), lambda: ops.quantize_int8(x[:, :0]),
            lambda: ops.quantize_weight_int8(q[0]), lambda: ops.quantize_weight_int8(x[:, :24]),
            lambda: ops.linear_int8(x, q8, s8), lambda: ops.linear_fp8(x, q, s), lambda: ops.linear_fp8(x, q, s8), lambda: ops.linear_int8(x, q, s[:63]), lambda: ops.linear_int8(x, q, s[None]),
            lambda: ops.linear_int8(x, q, s.double()), lambda: ops.linear_int8(x, q, None), lambda: ops.linear_int8(x, None, s), lambda: ops.linear_int8(x, q.T, s),
            lambda: ops.linear_int8(x, q[:, :120], s), lambda: ops.linear_int8(x[:, :64], q, s), lambda: ops.linear_int8(x, q, s, torch.zeros(64, device=device)),
            lambda: ops.linear_int8(x, q, s, torch.zeros(63, dtype=BF16, device=device)), lambda: ops.linear_int8(x, q, s, out_dtype=torch.float64),
            lambda: ops.linear_int8((x, s), q, s), lambda: ops.linear_int8((q, s8), q, s), lambda: ops.linear_int8((q8, s), q, s), lambda: ops.linear_int8((q, s[:3]), q, s),
            lambda: ops.linear_fp8(rows, q8, s8), lambda: ops.linear_int8((rows[0],), q, s), lambda: ops.linear_int8((rows[0], None), q, s),
            lambda: ops.linear_int8(x, torch.zeros(1, 1 << 17, dtype=I8, device=device), torch.zeros(1, device=device)),
            lambda: ops.linear_int8(torch.zeros(2, 128, dtype=torch.int32, device=device), q, s), lambda: ops.linear_int8(rows[0], q, s),
            lambda: ops.grouped_mm(rows, (q, s), ends), lambda: ops.grouped_mm(rows, (q[None], s), ends), lambda: ops.grouped_mm(rows, (q[None], s[None]), ends.long()),
            lambda: ops.grouped_mm(rows, (q8[None], s8[None]), ends), lambda: ops.grouped_mm((q8, torch.zeros(64, 1, device=device)), (q[None], s[None]), ends),
            lambda: ops.grouped_mm(rows, x[None], ends), lambda: ops.grouped_mm(rows, q[None], ends),
            lambda: moe(x, ids, p, gu, (dn[0].to(F32).to(E4M3), dn[1])), lambda: moe(x, ids, p, (gu[0], gu[1][:, :31]), dn), lambda: moe(x, ids, p, gu, dn[0]),
            lambda: moe(x, ids, p, (gu[0][..., :112], gu[1]), dn), lambda: moe(x, ids, p, (gu[0][:, :16], gu[1][:, :16]), dn), lambda: moe(x.float(), ids, p, gu, dn),
            lambda: moe(x, ids.float(), p, gu, dn)]


def test_refusals_without_a_gpu():
    x, w = torch.zeros(2, 128, dtype=BF16), torch.zeros(128, dtype=BF16)
    q, s = torch.zeros(64, 128, dtype=I8), torch.zeros(64)
    for call in (lambda: ops.rms_norm(x, w, quantize=I8), lambda: ops.quantize_int8(x), lambda: ops.linear_int8(x, q, s),
                 lambda: ops.grouped_mm((q, s), (q[None], s[None]), torch.zeros(1, dtype=torch.int32)),
                 lambda: ops.moe_experts_stacked(x, torch.zeros(2, 1, dtype=torch.int64), torch.zeros(2, 1), (q[None, :32], s[None, :32]), (torch.zeros(1, 128, 16, dtype=I8), torch.zeros(1, 128)))):
        with pytest.raises(RuntimeError, match="ROCm device only"):
            call()
    for k, call in enumerate(wrong_calls("cpu")):
        with pytest.raises(RuntimeError):
            call()
            pytest.fail(f"call {k} was taken")


@pytest.mark.gpu
def test_refusals_on_a_gpu(gen):
    for k, call in enumerate(wrong_calls("cuda")):
        with pytest.raises(RuntimeError):
            call()
            pytest.fail(f"call {k} was taken")
    x, (q, s) = randn(gen, 2, 128, dtype=BF16), weight(gen, 64, 128)
    ends = torch.ones(1, dtype=torch.int32, device="cuda")
    for call in (lambda: ops.linear_int8(x, q.cpu(), s), lambda: ops.linear_int8(x, q, s.cpu()), lambda: ops.grouped_mm(x, (q[None], s[None]), ends.cpu()),
                 lambda: ops.linear_int8((q, s.cpu()), q, s)):
        with pytest.raises(RuntimeError, match="device of x"):
            call()
    gu, dn = experts(gen, 1, 128, 128)
    ids, wt = torch.zeros(2, 1, dtype=torch.int64, device="cuda"), torch.ones(2, 1, device="cuda")
    leaf, asks = x.clone().requires_grad_(), lambda p: (p[0], p[1].clone().requires_grad_())
    for call in (lambda: ops.rms_norm(leaf, x[0], quantize=I8), lambda: ops.quantize_int8(leaf), lambda: ops.linear_int8(leaf, q, s), lambda: ops.linear_int8(x, *asks((q, s))),
                 lambda: ops.linear_int8(asks((q, s)), q, s), lambda: ops.grouped_mm(x, asks(gu), ends), lambda: ops.moe_experts_stacked(x, ids, wt, asks(gu), dn)):
        with pytest.raises(RuntimeError, match="no derivative"):
            call()
        with torch.no_grad():
            call()


def test_status_codes_without_a_gpu():
    L = _native.lib()
    p, odd = ctypes.c_void_p(0x1000), ctypes.c_void_p(0x1001)          # never dereferenced: every call below is refused first, or does nothing
    norm = lambda x=p, r=None, w=p, rows=1, n=128, dt=0, y=p, s=p, t=None: L.htr_rms_norm_int8(x, n, r, n, w, rows, n, 1e-6, dt, y, s, t, None)
    assert norm(rows=0) == 0 and norm(rows=-1) == 11 and norm(n=0) == 11 and norm(n=24) == 11 and norm(rows=1 << 31) == 11 and norm(dt=3) == 5 and norm(dt=4) == 5
    assert norm(x=None) == 1 and norm(r=p) == 1 and norm(t=p) == 1 and norm(y=None) == 1 and norm(s=None) == 1 and norm(x=odd) == 7 and norm(s=odd) == 7
    quant = lambda x=p, stride=128, rows=1, n=128, dt=0, q=p, s=p: L.htr_quantize_int8(x, stride, rows, n, dt, q, s, None)
    assert quant(rows=0) == 0 and quant(n=24) == 11 and quant(dt=4) == 5 and quant(q=None) == 1 and quant(x=odd) == 7 and quant(q=odd) == 7 and quant(n=(1 << 30) + 16) == 11
    prod = lambda x=p, xs=p, w=p, ws=p, b=None, ends=None, y=p, rows=1, m=128, n=128, E=1, xt=4, yt=0: \
        L.htr_product(x, xt, xs, w, ws, b, ends, y, rows, m, n, E, 4, yt, None)
    assert prod(rows=0) == 0 and prod(n=24) == 11 and prod(n=1 << 17) == 11 and prod(m=0) == 11 and prod(yt=4) == 5 and prod(xt=3) == 5 and prod(xt=2, ws=None) == 1 and prod(xt=2, rows=9) == 5 and prod(E=2) == 1
    assert prod(xs=None) == 1 and prod(ws=None) == 1 and prod(x=odd) == 7 and prod(w=odd) == 7 and prod(ws=odd) == 7 and prod(xs=odd) == 7
    # floating rows with an int8 matrix: few, that the product rounds itself, and one matrix
    floating = lambda xt, rows=1, n=128, ends=None, x=p: L.htr_product(x, xt, None, p, None, None, ends, p, rows, 64, n, 1, 4, 0, None)
    assert [L.htr_product_rounds_int8(*a) for a in ((1, 4096), (8, 4096), (9, 4096), (0, 4096), (1, 131056), (8, 14336), (8, 24576))] == [1, 1, 0, 0, 1, 1, 0]
    assert floating(0) == 1 and floating(2) == 1 and floating(3) == 5 and floating(0, rows=9) == 5 and floating(0, ends=p) == 5 and floating(1, rows=8, n=24576) == 5
    need = L.htr_moe_stacked_scratch_bytes
    assert need(4, 2, 8, 256, 128, 4) > 0 and need(4, 2, 8, 256, 72, 4) == 0 and need(4, 2, 8, 72, 128, 4) == 0 and need(4, 2, 8, 256, 80, 4) > 0 and need(4, 2, 8, 1 << 17, 128, 4) == 0
    a256 = ctypes.c_void_p(0x100000)
    moe = lambda dt=0, gus=p, sc=a256, bytes=1 << 30, T=4: L.htr_moe_stacked(p, dt, p, 1, p, T, 2, p, gus, p, gus, 8, 256, 128, 4, p, sc, bytes, None)
    assert moe(T=0) == 11 and moe(dt=2) == 5 and moe(gus=None) == 1 and moe(sc=None) == 6 and moe(bytes=100) == 6


# ---- the C++ host path and the Python one
@pytest.mark.gpu
def test_both_host_paths_agree(gen, monkeypatch):
    x, w = randn(gen, 5, 256, dtype=BF16), randn(gen, 256, dtype=BF16)
    r, b = randn(gen, 5, 256, dtype=BF16), randn(gen, 64, dtype=BF16)
    q, s = weight(gen, 64, 256)
    gu, dn = experts(gen, 3, 256, 144)
    ends = torch.tensor([2, 2, 4], dtype=torch.int32, device="cuda")
    ids, wt = torch.tensor([[0, 2], [1, 1], [2, 0], [0, 1], [2, 2]], device="cuda"), torch.rand(5, 2, device="cuda", generator=gen)
    xq = ops.quantize_int8(x)
    many = randn(gen, 40, 256, dtype=F16)
    calls = [lambda: ops.rms_norm(x, w, quantize=I8), lambda: ops.rms_norm(x, w, residual=r, quantize=I8), lambda: ops.linear_int8(x, q, s, b), lambda: ops.linear_int8(xq, q, s, out_dtype=F32),
             lambda: ops.linear_int8(x.float(), q, s), lambda: ops.linear_int8(many, q, s), lambda: ops.grouped_mm(xq, gu, ends), lambda: ops.grouped_mm(x, gu, ends, out_dtype=F16),
             lambda: ops.moe_experts_stacked(x, ids, wt, gu, dn)]
    flat = lambda o: [o] if isinstance(o, torch.Tensor) else [t for p in o for t in flat(p)]
    fast, taken = _native.fast(), []

    class Spy:
        def __getattr__(self, name):
            def call(*a):
                y = getattr(fast, name)(*a)
                taken.append((name, y is not None))
                return y
            return call

    for call in calls:
        monkeypatch.setattr(_native, "fast", Spy)
        taken.clear()
        got = flat(call())
        assert len(taken) == 1 and taken[0][1], taken                  # the C++ path took it
        monkeypatch.setattr(_native, "fast", lambda: None)
        want = flat(call())
        assert len(got) == len(want)
        for u, v in zip(got, want):
            assert u.dtype == v.dtype and u.shape == v.shape and torch.equal(u, v)
