"""The operators around the packed linears (ops.rms_norm, linear_fp8, grouped_mm, moe_experts_stacked) against their definitions in 64 bits.

Tolerances are bounds by arithmetic.  A rounding to type t is off by at most half a step, finfo(t).eps / 2 relative (and half the smallest subnormal).
A float32 sum of n products is off by at most n 2^-23 times the sum of the products' magnitudes, whatever the order and whether the matrix unit rounds
or cuts off its partial sums; the block scales of e4m3 rows add two more roundings to every block."""
import ctypes

import pytest
import torch

from htr_amd import _native, ops

BF16, F16, F32, E4M3 = torch.bfloat16, torch.float16, torch.float32, torch.float8_e4m3fn


@pytest.fixture
def gen():
    return torch.Generator(device="cuda").manual_seed(20261206)


def randn(gen, *shape, dtype=F32, scale=1.0):
    return (torch.randn(*shape, device=gen.device, generator=gen) * scale).to(dtype)


# ---- definitions
def half_step(y, dtype):
    """Largest error of rounding y to dtype."""
    f = torch.finfo(dtype)
    return y.abs() * (f.eps / 2) + f.smallest_normal * f.eps / 2


def to_e4m3(v):
    """Float64 to the nearest e4m3 value, ties to even; NaN stays."""
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(v / step) * step


def quantized(x):
    """(values, scales) of float64 rows."""
    b = x.unflatten(-1, (-1, 128))
    b = torch.where(b.isfinite(), b, torch.nan)
    amax = b.abs().nan_to_num(0.0).amax(-1).clamp(min=2.0 ** -100)
    e = torch.floor(torch.log2(amax / 448))
    s = torch.exp2(e)
    for _ in range(2):
        s = torch.where(s * 448 < amax, s * 2, s)
    s = torch.where(s * 224 >= amax, s / 2, s)
    return to_e4m3(b / s[..., None]).flatten(-2), s


def value(q, s):
    """Float64 values of 8-bit rows or matrices."""
    s = s.double().repeat_interleave(128, -1)
    if s.shape != q.shape:
        s = s.repeat_interleave(128, -2)[..., :q.shape[-2], :]
    return q.double() * s


def assert_within(got, want, bound):
    got = got.double()
    assert got.shape == want.shape
    assert torch.equal(got.isnan(), want.isnan())
    off = ((got - want).abs() - bound).nan_to_num(0.0)
    assert off.max().item() <= 0 if off.numel() else True, f"{off.max().item()} beyond the bound at {off.argmax().item()}"


def product_bound(x, w, dtype, bias=None):
    """(y, bound) of x @ w^T (+ bias) in float32 sums, rounded to dtype."""
    y, mag = x @ w.T, x.abs() @ w.abs().T
    bound = mag * (x.shape[1] * 2.0 ** -23 + 4 * 2.0 ** -24)
    if bias is not None:
        y = y + bias.double()
        bound = bound + y.abs() * 2.0 ** -24
    return y, bound * 1.01 + half_step(y.abs() + bound, dtype)


def fp8_weight(gen, *shape):
    """An 8-bit matrix whose scales are not powers of two."""
    q, s = ops.quantize_weight_fp8(randn(gen, *shape, scale=shape[-1] ** -0.5))
    return q, s * (0.5 + torch.rand(s.shape, device=s.device, generator=gen))


# ---- norm
def norm64(x, w, eps, residual):
    t = x if residual is None else (x.float() + residual.float()).to(x.dtype)
    d = t.double()
    return d / torch.sqrt((d * d).mean(-1, keepdim=True) + eps) * w.double(), t


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("rows,n", [(1, 1), (1, 4096), (3, 7), (5, 64), (2, 130), (17, 520), (4, 2824), (3, 8192), (2, 8200), (2, 16384), (1, 32768), (1, 40000)])
@pytest.mark.parametrize("residual", [False, True])
def test_norm(gen, dtype, rows, n, residual):
    x, w = randn(gen, rows, n, dtype=dtype), randn(gen, n, dtype=dtype)
    r = randn(gen, rows, n, dtype=dtype, scale=3) if residual else None
    y = ops.rms_norm(x, w, 1e-5, residual=r)
    want, t = norm64(x, w, 1e-5, r)
    if residual:
        y, total = y
        assert torch.equal(total, t)
    # the root in 64 bits rounded to float32, two products: three roundings
    assert_within(y, want, want.abs() * 3.01 * 2.0 ** -24 + half_step(want * (1 + 2.0 ** -22), dtype))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("rows,n", [(1, 128), (1, 4096), (7, 384), (33, 1408), (3, 8192), (2, 8320), (2, 16384), (1, 40960)])
@pytest.mark.parametrize("residual", [False, True])
def test_norm_in_eight_bits(gen, dtype, rows, n, residual):
    x, w = randn(gen, rows, n, dtype=dtype), randn(gen, n, dtype=dtype)
    r = randn(gen, rows, n, dtype=dtype, scale=3) if residual else None
    out = ops.rms_norm(x, w, 1e-6, residual=r, quantize=True)
    want, t = norm64(x, w, 1e-6, r)
    if residual:
        out, total = out
        assert torch.equal(total, t)
    q, s = out
    assert q.dtype == E4M3 and s.dtype == F32 and s.shape == (rows, n // 128)
    assert torch.equal(s.double(), quantized(want)[1])
    # e4m3: half a step of 2^-3 relative, of 2^-9 below 2^-6; what is rounded is a float32 itself
    v = (want / s.double().repeat_interleave(128, -1)).abs()
    step = torch.exp2(torch.floor(torch.log2(v.clamp(min=2.0 ** -6))) - 3)
    assert_within(q, want / s.double().repeat_interleave(128, -1), step / 2 + v * 2.0 ** -23)


@pytest.mark.gpu
def test_norm_of_zeros_infinities_and_nan(gen):
    x = randn(gen, 4, 256, dtype=BF16)
    x[0] = 0
    x[1, 3] = float("inf")
    x[2, 200] = float("nan")
    w = torch.ones(256, dtype=BF16, device="cuda")
    y = ops.rms_norm(x, w)
    assert torch.equal(y[0], torch.zeros_like(y[0])) and y[1, 3].isnan() and (y[1, :3] == 0).all() and y[2].isnan().all() and y[3].isfinite().all()
    q, s = ops.rms_norm(x, w, quantize=True)
    assert (q[0].float() == 0).all() and (s[0] == 2.0 ** -108).all()
    assert q[1, 3].float().isnan() and (q[1, :3].float() == 0).all() and q[2].float().isnan().all() and s.isfinite().all()
    assert torch.equal(q[3].float(), ops.rms_norm(x[3:], w, quantize=True)[0][0].float())


@pytest.mark.gpu
@pytest.mark.parametrize("n", [256, 40960])
@pytest.mark.parametrize("dtype,size,weight", [(F32, 1e38, 1.0), (F32, 1e-39, 1.0), (F32, 1e30, 1e20), (BF16, 2.0 ** 125, 1.0), (BF16, 2.0 ** 124, 2.0 ** 20),
                                               (BF16, 2.0 ** -100, 2.0 ** -40), (F16, 2.0 ** -12, 2.0 ** -12)])
def test_norm_of_rows_of_any_size(gen, dtype, n, size, weight):
    """Factors, or products with the weight, that float32 cannot hold, of results that it can."""
    sign = lambda: torch.randint(0, 2, (3, n), device="cuda", generator=gen) * 2 - 1
    x = (sign() * size * (1 + torch.rand(3, n, device="cuda", generator=gen))).to(dtype)
    w = (weight * (1 + torch.rand(n, device="cuda", generator=gen))).to(dtype)
    assert x.isfinite().all()
    want, _ = norm64(x, w, 0.0, None)
    # as in test_norm; below the smallest normal value a rounding in float32 is off by half of 2^-149
    assert_within(ops.rms_norm(x, w, 0.0), want, want.abs() * 3.01 * 2.0 ** -24 + 2.0 ** -149 + half_step(want * (1 + 2.0 ** -22), dtype))
    q, s = ops.rms_norm(x, w, 0.0, quantize=True)
    assert torch.equal(s.double(), quantized(want)[1])
    v = (want / s.double().repeat_interleave(128, -1)).abs()                               # as in test_norm_in_eight_bits
    step = torch.exp2(torch.floor(torch.log2(v.clamp(min=2.0 ** -6))) - 3)
    assert_within(q, want / s.double().repeat_interleave(128, -1), step / 2 + v * 2.0 ** -23)


@pytest.mark.gpu
@pytest.mark.parametrize("quantize", [False, True])
def test_norm_takes_strides_and_any_alignment(gen, quantize):
    big, w = randn(gen, 6, 3, 400, dtype=BF16), randn(gen, 257, dtype=BF16)
    for x in (big[:, 1, 5:261], big[::2, :, 8:264], big[:, :, 0:256].transpose(0, 1), big.transpose(1, 2)[:, :256, :2].transpose(1, 2)):
        for weight in (w[:256], w[1:]):
            r = randn(gen, *x.shape, dtype=BF16)
            got = ops.rms_norm(x, weight, residual=r, quantize=quantize)
            want = ops.rms_norm(x.contiguous(), weight.clone(), residual=r, quantize=quantize)
            flat = lambda o: (*o[0], o[1]) if quantize else o
            for a, b in zip(flat(got), flat(want)):
                assert torch.equal(a.float(), b.float())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("n", [640, 1027, 8192, 8320])
@pytest.mark.parametrize("residual", [False, True])
def test_norm_of_many_rows(gen, dtype, n, residual):
    x, w = randn(gen, 2051, n, dtype=dtype), randn(gen, n, dtype=dtype)
    r = randn(gen, 2051, n, dtype=dtype, scale=3) if residual else None
    want, t = norm64(x, w, 1e-5, r)
    y = ops.rms_norm(x, w, 1e-5, residual=r)
    if residual:
        y, total = y
        assert torch.equal(total, t)
    assert_within(y, want, want.abs() * 3.01 * 2.0 ** -24 + half_step(want * (1 + 2.0 ** -22), dtype))            # as in test_norm
    if n % 128 == 0:
        q, s = ops.rms_norm(x, w, 1e-5, residual=r, quantize=True)[0] if residual else ops.rms_norm(x, w, 1e-5, quantize=True)
        assert torch.equal(s.double(), quantized(want)[1])
        v = (want / s.double().repeat_interleave(128, -1)).abs()                                                    # as in test_norm_in_eight_bits
        step = torch.exp2(torch.floor(torch.log2(v.clamp(min=2.0 ** -6))) - 3)
        assert_within(q, want / s.double().repeat_interleave(128, -1), step / 2 + v * 2.0 ** -23)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("n", [5, 9, 513, 1001, 8191, 8193, 16391, 32767, 32769])
def test_norm_of_rows_that_end_inside_a_run(gen, dtype, n):
    """Odd widths, odd distances from row to row, nothing on a 16-byte boundary; what lies around the rows is not read into them."""
    big = torch.full((4, n + 4), float("nan"), dtype=dtype, device="cuda")
    x, w = big[:, 3:n + 3], torch.full((n + 2,), float("nan"), dtype=dtype, device="cuda")
    x.copy_(randn(gen, 4, n))
    w[1:-1] = randn(gen, n)
    r = randn(gen, 4, n, dtype=dtype, scale=3)
    for residual in (None, r):
        y = ops.rms_norm(x, w[1:-1], 1e-5, residual=residual)
        want, t = norm64(x, w[1:-1], 1e-5, residual)
        if residual is not None:
            y, total = y
            assert torch.equal(total, t)
        assert_within(y, want, want.abs() * 3.01 * 2.0 ** -24 + half_step(want * (1 + 2.0 ** -22), dtype))     # as in test_norm


@pytest.mark.gpu
def test_norm_of_nothing():
    x, w = torch.empty(0, 128, device="cuda", dtype=BF16), torch.ones(128, device="cuda", dtype=BF16)
    assert ops.rms_norm(x, w).shape == (0, 128)
    (q, s), t = ops.rms_norm(x, w, residual=x, quantize=True)
    assert q.shape == t.shape == (0, 128) and s.shape == (0, 1)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_rows_to_eight_bits(gen, dtype):
    x = randn(gen, 37, 640, dtype=dtype) * torch.exp(4 * randn(gen, 37, 1)).to(dtype)
    x[3, 128:256] = 0
    x[4, 5], x[5, 600] = float("inf"), float("nan")
    x[6, 0:128] = 0
    x[6, 7] = 448 * 2.0 ** 3       # right at the border of a scale
    q, s = ops.quantize_fp8(x)
    want, scales = quantized(x.double())
    assert torch.equal(s.double(), scales) and s[6, 0] == 8
    assert torch.equal(q.double().nan_to_num(9e9), want.nan_to_num(9e9))          # the division is exact: one rounding


def test_weights_to_eight_bits():
    w = torch.randn(3, 200, 256, generator=torch.Generator().manual_seed(1))
    w[1, 130, 7] = float("inf")
    q, s = ops.quantize_weight_fp8(w)
    assert q.shape == w.shape and s.shape == (3, 2, 2) and s.isfinite().all() and q[1, 130, 7].float().isnan()
    w[1, 130, 7] = 0
    back = ops.dequantize_fp8(*ops.quantize_weight_fp8(w))
    assert ((back - w).abs() <= w.abs() * 2.0 ** -4 + s.amax() * 2.0 ** -10).all()


# ---- products
@pytest.mark.gpu
@pytest.mark.parametrize("m,n", [(1, 128), (100, 256), (128, 640), (384, 4096), (1030, 1152)])
@pytest.mark.parametrize("rows", [1, 2, 16, 17, 33, 64, 65, 100, 193, 300])
def test_linear_fp8(gen, m, n, rows):
    w, ws = fp8_weight(gen, m, n)
    for dtype, bias in ((BF16, False), (F16, True), (F32, True)):
        x = randn(gen, rows, n, dtype=dtype)
        b = randn(gen, m, dtype=dtype) if bias else None
        want, bound = product_bound(value(*quantized(x.double())), value(w, ws), dtype, b)
        y = ops.linear_fp8(x, w, ws, b)
        assert y.dtype == dtype
        assert_within(y, want, bound)
        q, s = ops.quantize_fp8(x)
        assert torch.equal(ops.linear_fp8((q, s), w, ws, b, out_dtype=dtype), y)        # rounded ahead or on the way: the same values and sums
    # scales of rows from elsewhere
    s = s * (0.5 + torch.rand(s.shape, device="cuda", generator=gen))
    want, bound = product_bound(value(q, s), value(w, ws), BF16)
    assert_within(ops.linear_fp8((q, s), w, ws), want, bound)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [3, 90, 260])
def test_a_row_with_nan_keeps_to_itself(gen, rows):
    w, ws = fp8_weight(gen, 144, 512)
    x = randn(gen, rows, 512, dtype=BF16)
    clean = ops.linear_fp8(x, w, ws)
    x[1, 5] = float("nan")
    x[2, 300] = float("-inf")
    y = ops.linear_fp8(x, w, ws)
    assert y[1:3].isnan().all()
    assert torch.equal(y[0], clean[0]) and torch.equal(y[3:], clean[3:])


@pytest.mark.gpu
def test_linear_fp8_takes_any_leading_dimensions(gen):
    w, ws = fp8_weight(gen, 96, 256)
    x = randn(gen, 2, 5, 300, dtype=BF16)[..., 3:259]
    y = ops.linear_fp8(x, w, ws)
    assert y.shape == (2, 5, 96)
    assert torch.equal(y.reshape(10, 96), ops.linear_fp8(x.reshape(10, 256).contiguous(), w, ws))
    assert ops.linear_fp8(x[:, :0], w, ws).shape == (2, 0, 96)
    assert torch.equal(ops.linear_fp8(x[0, 0], w, ws), y[0, 0])


def _ends(counts):
    return torch.tensor(counts, dtype=torch.int32).cumsum(0).to(torch.int32).cuda()


COUNTS = [[1], [0, 1, 0], [5, 0, 0, 11, 1], [16, 17, 0, 33, 1, 64], [0, 0, 0], [200, 0, 1, 130, 129], [300, 5], [3] * 70, [0] * 64 + [7, 0, 40]]


@pytest.mark.gpu
@pytest.mark.parametrize("counts", COUNTS, ids=lambda c: f"{len(c)}x{sum(c)}")
@pytest.mark.parametrize("kind", [BF16, F16, E4M3], ids=str)
@pytest.mark.parametrize("m,n", [(200, 256), (24, 1152)])
@pytest.mark.parametrize("behind", [0, 19])
def test_grouped_mm(gen, counts, kind, m, n, behind):
    R, E = sum(counts) + behind, len(counts)
    if kind == E4M3:
        x, w = ops.quantize_fp8(randn(gen, R, n)), fp8_weight(gen, E, m, n)
        xd, wd, dtype = value(*x), value(*w), BF16
    else:
        n -= 8 * (m % 3)             # a row that ends inside its last 128 bytes
        x, w = randn(gen, R, n, dtype=kind), randn(gen, E, m, n, dtype=kind, scale=n ** -0.5)
        xd, wd, dtype = x.double(), w.double(), kind
    y = ops.grouped_mm(x, w, _ends(counts))
    assert y.dtype == dtype and y.shape == (R, m)
    first = 0
    for e, c in enumerate(counts):
        want, bound = product_bound(xd[first:first + c], wd[e], dtype)
        assert_within(y[first:first + c], want, bound)
        first += c
    assert (y[first:] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [BF16, E4M3], ids=str)
@pytest.mark.parametrize("counts,m", [([e * 7 % 37 for e in range(130)], 512), ([2000, 0, 3100], 4096), ([0] * 63 + [1900, 0, 2500] + [1] * 70, 1000),
                                      ([300 - 4 * e for e in range(75)], 1024), ([0] * 64 + [700], 2900)], ids=lambda c: str(len(c) if isinstance(c, list) else c))
def test_grouped_mm_of_more_tiles_than_run_at_once(gen, kind, counts, m):
    """More than 64 experts, several tiles to a workgroup, every height of tile."""
    n, behind = 256, 45
    R, E = sum(counts) + behind, len(counts)
    if kind == E4M3:
        x, w = ops.quantize_fp8(randn(gen, R, n)), fp8_weight(gen, E, m, n)
        xd, wd = value(*x), w
    else:
        x, w = randn(gen, R, n, dtype=kind), randn(gen, E, m, n, dtype=kind, scale=n ** -0.5)
        xd, wd = x.double(), w
    ends = _ends(counts)
    y = ops.grouped_mm(x, w, ends)
    first = 0
    for e, c in enumerate(counts):
        if c:
            want, bound = product_bound(xd[first:first + c], value(wd[0][e], wd[1][e]) if kind == E4M3 else wd[e].double(), BF16)
            assert_within(y[first:first + c], want, bound)
        first += c
    assert (y[first:] == 0).all()
    wild = ends.clone()
    wild[0::3] -= 2 ** 30                      # each counts as the one before it
    meant = wild.clamp(0, R).cummax(0).values.int()
    assert torch.equal(ops.grouped_mm(x, w, wild), ops.grouped_mm(x, w, meant))


@pytest.mark.gpu
@pytest.mark.parametrize("n", [8, 24, 56, 64, 72, 120, 136, 1000])
@pytest.mark.parametrize("counts", [[3, 1], [100, 90], [300, 400]])
def test_grouped_mm_on_short_rows(gen, n, counts):
    """Rows that end at any multiple of 16 bytes; what lies behind them in memory is NaN."""
    R = sum(counts)
    room = torch.full((R * n + 64,), float("nan"), dtype=BF16, device="cuda")
    x = room[:R * n].view(R, n)
    x.copy_(randn(gen, R, n, dtype=BF16))
    room2 = torch.full((2 * 40 * n + 64,), float("nan"), dtype=BF16, device="cuda")
    w = room2[:2 * 40 * n].view(2, 40, n)
    w.copy_(randn(gen, 2, 40, n, dtype=BF16))
    y = ops.grouped_mm(x, w, _ends(counts), out_dtype=F32)
    for e, rows in enumerate((slice(0, counts[0]), slice(counts[0], R))):
        want, bound = product_bound(x[rows].double(), w[e].double(), F32)
        assert_within(y[rows], want, bound)


@pytest.mark.gpu
@pytest.mark.parametrize("ends,meant", [([4, 2, 9], [4, 4, 9]), ([-5, 3, 100], [0, 3, 40]), ([2 ** 31 - 1, 0, 7], [40, 40, 40]), ([-1, -2, -3], [0, 0, 0])])
def test_ends_out_of_order_or_range(gen, ends, meant):
    x, w = randn(gen, 40, 64, dtype=BF16), randn(gen, 3, 48, 64, dtype=BF16)
    got = ops.grouped_mm(x, w, torch.tensor(ends, dtype=torch.int32, device="cuda"))
    assert torch.equal(got, ops.grouped_mm(x, w, torch.tensor(meant, dtype=torch.int32, device="cuda")))
    assert (got[meant[-1]:] == 0).all()


# ---- routed experts
def moe64(x, ids, wt, gate_up, down, eight, dtype):
    """(y, bound) of the layer with its roundings; the bound follows what float32 sums may make of each hidden value before it is rounded."""
    T, H = x.shape
    xd = value(*quantized(x.double())) if eight else x.double()
    gu = value(*gate_up) if eight else gate_up.double()
    dn = value(*down) if eight else down.double()
    F = dn.shape[2]
    y, bound = torch.zeros(T, H, dtype=torch.float64, device=x.device), torch.zeros(T, H, dtype=torch.float64, device=x.device)
    silu = lambda g: g / (1 + torch.exp(-g))
    for j in range(ids.shape[1]):
        for t in range(T):
            e = int(ids[t, j])
            if not 0 <= e < gu.shape[0]:
                y[t] = float("nan")
                continue
            g, mag = gu[e] @ xd[t], gu[e].abs() @ xd[t].abs()
            off = mag * (H * 2.0 ** -23 + 2.0 ** -21)
            corners = torch.stack([silu(g[:F] + a * off[:F]) * (g[F:] + b * off[F:]) for a in (-1, 1) for b in (-1, 1)])
            h = silu(g[:F]) * g[F:]
            slack = h.abs() * 2.0 ** -20                                   # exp and three float32 operations
            lo, hi = torch.minimum(corners.amin(0), h) - slack, torch.maximum(corners.amax(0), h) + slack
            if eight:
                q, s = quantized(h)
                s = s.repeat_interleave(128)
                h, lo, hi = q * s, to_e4m3(lo / s) * s, to_e4m3(hi / s) * s
                room = torch.maximum(hi - h, h - lo) + s * 2.0 ** -9       # another scale: another subnormal step
            else:
                lo, hi = lo - half_step(lo, dtype), hi + half_step(hi, dtype)
                room = torch.maximum(hi - h, h - lo)
            w = wt[t, j].double()
            out, away = dn[e] @ h, dn[e].abs() @ room
            away = away + (dn[e].abs() @ (h.abs() + room)) * (F * 2.0 ** -23 + 2.0 ** -21)
            y[t] += w * out
            bound[t] += w.abs() * away + (w * out).abs() * 2.0 ** -20
    return y, bound * 1.01 + half_step(y.abs() + bound, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("eight", [False, True], ids=["16", "8"])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("T,E,top,H,F", [(1, 4, 2, 256, 128), (5, 8, 3, 128, 384), (40, 3, 1, 256, 256), (9, 70, 8, 128, 128), (70, 2, 2, 384, 128)])
def test_moe_experts_stacked(gen, eight, dtype, T, E, top, H, F):
    x = randn(gen, T, H, dtype=dtype)
    ids = torch.argsort(torch.rand(T, E, device="cuda", generator=gen))[:, :top]
    wt = torch.rand(T, top, device="cuda", generator=gen)
    if eight:
        gate_up, down = fp8_weight(gen, E, 2 * F, H), fp8_weight(gen, E, H, F)
    else:
        gate_up, down = randn(gen, E, 2 * F, H, dtype=dtype, scale=H ** -0.5), randn(gen, E, H, F, dtype=dtype, scale=F ** -0.5)
    y = ops.moe_experts_stacked(x, ids, wt, gate_up, down)
    assert y.dtype == dtype
    want, bound = moe64(x, ids, wt, gate_up, down, eight, dtype)
    assert_within(y, want, bound)
    assert torch.equal(ops.moe_experts_stacked(x, ids.int(), wt.double(), gate_up, down), y)
    assert torch.equal(ops.moe_experts_stacked(x, ids, wt, gate_up, down), y)


@pytest.mark.gpu
@pytest.mark.parametrize("eight", [False, True], ids=["16", "8"])
def test_moe_of_more_experts_than_a_wave_has_lanes(gen, eight):
    T, E, top, H, F, dtype = 60, 70, 7, 256, 128, BF16
    x, wt = randn(gen, T, H, dtype=dtype), torch.rand(T, top, device="cuda", generator=gen)
    ids = torch.argsort(torch.rand(T, E, device="cuda", generator=gen))[:, :top]
    if eight:
        gate_up, down = fp8_weight(gen, E, 2 * F, H), fp8_weight(gen, E, H, F)
    else:
        gate_up, down = randn(gen, E, 2 * F, H, dtype=dtype, scale=H ** -0.5), randn(gen, E, H, F, dtype=dtype, scale=F ** -0.5)
    assert_within(ops.moe_experts_stacked(x, ids, wt, gate_up, down), *moe64(x, ids, wt, gate_up, down, eight, dtype))


@pytest.mark.gpu
@pytest.mark.parametrize("eight", [False, True], ids=["16", "8"])
def test_moe_with_one_expert_twice_and_experts_out_of_range(gen, eight):
    T, E, H, F = 6, 4, 256, 128
    x = randn(gen, T, H, dtype=BF16)
    ids = torch.randint(0, E, (T, 3), device="cuda", generator=gen)
    ids[0] = 2
    ids[1, 1], ids[2, 0], ids[3, 2] = -1, E, 2 ** 40
    wt = torch.rand(T, 3, device="cuda", generator=gen)
    if eight:
        gate_up, down = fp8_weight(gen, E, 2 * F, H), fp8_weight(gen, E, H, F)
    else:
        gate_up, down = randn(gen, E, 2 * F, H, dtype=BF16, scale=H ** -0.5), randn(gen, E, H, F, dtype=BF16, scale=F ** -0.5)
    want, bound = moe64(x, ids, wt, gate_up, down, eight, BF16)
    y = ops.moe_experts_stacked(x, ids, wt, gate_up, down)
    assert y[1:4].isnan().all()
    assert_within(y, want, bound)
    assert ops.moe_experts_stacked(x, torch.full_like(ids, -1), wt, gate_up, down).isnan().all()
    assert ops.moe_experts_stacked(x[:0], ids[:0], wt[:0], gate_up, down).shape == (0, H)
    assert (ops.moe_experts_stacked(x, ids[:, :0], wt[:, :0], gate_up, down) == 0).all()


# ---- as they are used
def _block(gen, H=256, F=128, E=6):
    """A decoder block's tail: norm, an 8-bit linear, norm, routed experts."""
    wt = dict(n1=randn(gen, H, dtype=BF16), o=fp8_weight(gen, H, H), n2=randn(gen, H, dtype=BF16), router=randn(gen, E, H, scale=H ** -0.5),
              gate_up=fp8_weight(gen, E, 2 * F, H), down=fp8_weight(gen, E, H, F))

    def run(x, h):
        xq, h = ops.rms_norm(x, wt["n1"], residual=h, quantize=True)
        y = ops.linear_fp8(xq, *wt["o"])
        y, h = ops.rms_norm(y, wt["n2"], residual=h)
        p, ids = torch.topk(torch.softmax(y.float() @ wt["router"].T, -1), 2, dim=-1)
        return ops.moe_experts_stacked(y, ids, p, wt["gate_up"], wt["down"]), h
    return run


@pytest.mark.gpu
def test_a_block_of_them_eager_on_streams_and_captured(gen):
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


@pytest.mark.gpu
def test_beyond_32_bits(gen):
    """Matrices, rows and results whose places in memory pass 2^32 bytes."""
    E, m, n = 40, 8192, 16384
    w = torch.zeros(E, m, n, dtype=torch.uint8, device="cuda").view(E4M3)              # 5.4 GB
    ws = torch.zeros(E, m // 128, n // 128, device="cuda")
    q, s = fp8_weight(gen, 256, n)
    w[E - 1, m - 256:], ws[E - 1, m // 128 - 2:] = q, s
    ends = torch.zeros(E, dtype=torch.int32, device="cuda")
    for rows in (3, 200):
        ends[E - 1] = rows
        x = ops.quantize_fp8(randn(gen, rows, n))
        want, bound = product_bound(value(*x), value(q, s), BF16)
        y = ops.grouped_mm(x, (w, ws), ends)
        assert_within(y[:, m - 256:], want, bound)
        assert (y[:, :m - 256] == 0).all()
    del w, ws
    rows, n = 1_200_000, 128
    x, q, s = randn(gen, rows, n, dtype=BF16), *fp8_weight(gen, 2048, n)
    y = ops.linear_fp8(x, q, s)                                                        # 4.9 GB
    last = slice(rows - 5, rows)
    assert torch.equal(y[last], ops.linear_fp8(x[last].clone(), q, s))
    y = ops.rms_norm(y, torch.ones(2048, dtype=BF16, device="cuda"), residual=y)[0]
    tail = ops.linear_fp8(x[last].clone(), q, s)
    assert torch.equal(y[last], ops.rms_norm(tail, torch.ones(2048, dtype=BF16, device="cuda"), residual=tail)[0])


@pytest.mark.gpu
def test_more_rows_than_a_launch_takes(gen):
    rows = (1 << 21) + 3
    x, w = randn(gen, rows, 128, dtype=BF16), randn(gen, 128, dtype=BF16)
    for a, b in zip(ops.rms_norm(x, w, quantize=True), ops.rms_norm(x[rows - 7:].clone(), w, quantize=True)):
        assert torch.equal(a[rows - 7:].float(), b.float())
    assert torch.equal(ops.rms_norm(x[:, 1:], w[1:], residual=x[:, 1:])[0][rows - 7:], ops.rms_norm(x[rows - 7:, 1:].clone(), w[1:].clone(), residual=x[rows - 7:, 1:].clone())[0])


@pytest.mark.gpu
def test_under_torch_compile(gen):
    run = _block(gen)
    x, h = randn(gen, 9, 256, dtype=BF16), randn(gen, 9, 256, dtype=BF16)
    got = torch.compile(run, backend="eager")(x, h)
    for a, b in zip(got, run(x, h)):
        assert torch.equal(a, b)


# ---- refusals
def test_refusals_without_a_gpu():
    x, w = torch.zeros(2, 128, dtype=BF16), torch.zeros(128, dtype=BF16)
    q, s = torch.zeros(64, 128).to(E4M3), torch.zeros(1, 1)
    ends = torch.zeros(1, dtype=torch.int32)
    bad = pytest.raises(RuntimeError)
    for call in (lambda: ops.rms_norm(x, w), lambda: ops.linear_fp8(x, q, s), lambda: ops.grouped_mm(x, x[None], ends), lambda: ops.quantize_fp8(x),
                 lambda: ops.moe_experts_stacked(x, torch.zeros(2, 1, dtype=torch.int64), torch.zeros(2, 1), torch.zeros(1, 16, 128, dtype=BF16),
                                                 torch.zeros(1, 128, 8, dtype=BF16))):
        with pytest.raises(RuntimeError, match="ROCm device only"):
            call()
    for call in (lambda: ops.rms_norm(x, w.float()), lambda: ops.rms_norm(x, w[:64]), lambda: ops.rms_norm(x.double(), w.double()),
                 lambda: ops.rms_norm(x, w, residual=x[:1]), lambda: ops.rms_norm(x[:, :100], w[:100], quantize=True),
                 lambda: ops.rms_norm(x, w, residual=x.float()), lambda: ops.rms_norm(x[:, :0], w[:0]),
                 lambda: ops.quantize_fp8(x[:, :64]), lambda: ops.quantize_fp8(x.double()),
                 lambda: ops.linear_fp8(x, q, s[:, :0]), lambda: ops.linear_fp8(x, q.float(), s), lambda: ops.linear_fp8(x[:, :64], q, s),
                 lambda: ops.linear_fp8(x, q, s, torch.zeros(64)), lambda: ops.linear_fp8(x, q, s, torch.zeros(63, dtype=BF16)),
                 lambda: ops.linear_fp8(x, q, s, out_dtype=torch.float64), lambda: ops.linear_fp8(x, q.T, s),
                 lambda: ops.linear_fp8((x, s), q, s), lambda: ops.linear_fp8((q, s), q, s),
                 lambda: ops.grouped_mm(x, x[None].half(), ends), lambda: ops.grouped_mm(x, x[None], ends.long()),
                 lambda: ops.grouped_mm(x, x[None], torch.zeros(2, dtype=torch.int32)), lambda: ops.grouped_mm(x[:, :60], x[None, :, :60], ends),
                 lambda: ops.grouped_mm(x, x[None].transpose(1, 2), ends), lambda: ops.grouped_mm(x[0], x[None], ends),
                 lambda: ops.moe_experts_stacked(x, ends[None], ends[None], x[None], x[None])):
        with bad:
            call()


@pytest.mark.gpu
def test_refusals_on_a_gpu(gen):
    x, w = randn(gen, 2, 128, dtype=BF16), randn(gen, 128, dtype=BF16)
    q, s = fp8_weight(gen, 64, 128)
    ids, wt = torch.zeros(2, 1, dtype=torch.int64, device="cuda"), torch.ones(2, 1, device="cuda")
    gu, dn = randn(gen, 1, 16, 128, dtype=BF16), randn(gen, 1, 128, 8, dtype=BF16)
    ends = torch.ones(1, dtype=torch.int32, device="cuda")
    for call in (lambda: ops.rms_norm(x, w.cpu()), lambda: ops.rms_norm(x, w, residual=x.cpu()), lambda: ops.linear_fp8(x, q.cpu(), s),
                 lambda: ops.linear_fp8(x, q, s.cpu()), lambda: ops.grouped_mm(x, x[None], ends.cpu()),
                 lambda: ops.moe_experts_stacked(x, ids.cpu(), wt, gu, dn)):
        with pytest.raises(RuntimeError, match="device of x"):
            call()
    leaf = x.clone().requires_grad_()
    for call in (lambda: ops.rms_norm(leaf, w), lambda: ops.linear_fp8(leaf, q, s), lambda: ops.grouped_mm(leaf, x[None], ends),
                 lambda: ops.moe_experts_stacked(x, ids, wt.clone().requires_grad_(), gu, dn), lambda: ops.quantize_fp8(leaf)):
        with pytest.raises(RuntimeError, match="no derivative"):
            call()
        with torch.no_grad():
            call()
    gu8, dn8 = fp8_weight(gen, 1, 256, 128), fp8_weight(gen, 1, 128, 128)
    asks = lambda p: (p[0].clone().requires_grad_(), p[1])
    for call in (lambda: ops.linear_fp8(x, *asks((q, s))), lambda: ops.linear_fp8(asks(ops.quantize_fp8(x)), q, s), lambda: ops.grouped_mm(x, asks(gu8), ends),
                 lambda: ops.moe_experts_stacked(x, ids, wt, asks(gu8), dn8), lambda: ops.moe_experts_stacked(x, ids, wt, gu8, asks(dn8))):
        with pytest.raises(RuntimeError, match="no derivative"):
            call()
    with pytest.raises(RuntimeError, match="ends must be int32"):
        ops.grouped_mm(x, x[None], None)


def test_status_codes_without_a_gpu():
    L = _native.lib()
    p, odd = ctypes.c_void_p(0x1000), ctypes.c_void_p(0x1001)          # never dereferenced: every call below is refused first, or does nothing
    norm = lambda x=p, r=None, w=p, rows=1, n=128, dt=0, y=p, s=None, t=None: L.htr_rms_norm(x, n, r, n, w, rows, n, 1e-6, dt, y, s, t, None)
    assert norm(rows=0) == 0 and norm(rows=-1) == 11 and norm(n=0) == 11 and norm(rows=1 << 31) == 11 and norm(dt=3) == 5
    assert norm(x=None) == 1 and norm(r=p) == 1 and norm(t=p) == 1 and norm(y=None) == 1 and norm(x=odd) == 7 and norm(n=100, s=p) == 11
    quant = lambda x=p, stride=128, rows=1, n=128, dt=0, q=p, s=p: L.htr_quantize_e4m3(x, stride, rows, n, dt, q, s, None)
    assert quant(rows=0) == 0 and quant(n=64) == 11 and quant(dt=3) == 5 and quant(q=None) == 1 and quant(x=odd) == 7 and quant(stride=129) == 7
    prod = lambda x=p, xs=p, w=p, ws=p, b=None, ends=None, y=p, rows=1, m=128, n=128, E=1, t=3, yt=0: \
        L.htr_product(x, t, xs, w, ws, b, ends, y, rows, m, n, E, t, yt, None)
    assert prod(rows=0) == 0 and prod(rows=-1) == 11 and prod(m=0) == 11 and prod(n=64) == 11 and prod(n=4, t=0) == 11 and prod(t=2) == 5 and prod(yt=3) == 5
    assert prod(E=2) == 1 and prod(E=0, ends=p) == 11 and prod(xs=None) == 1 and prod(ws=None) == 1 and prod(w=None) == 1 and prod(x=odd) == 7 and prod(y=odd) == 7
    assert prod(ends=odd) == 7 and prod(b=odd) == 7 and prod(rows=1 << 31) == 11 and prod(E=70000, ends=p) == 11
    assert prod(n=(1 << 22) + 128) == 11 and prod(m=(1 << 26) + 1) == 11 and quant(n=(1 << 30) + 128) == 11 and norm(n=(1 << 30) + 8) == 11         # places in a tile, and a launch, in 32 bits
    mixed = lambda xt, rows=1, t=3, xs=None: L.htr_product(p, xt, xs, p, None, None, None, p, rows, 128, 128, 1, t, 0, None)
    assert mixed(2) == 5 and mixed(0, rows=17) == 5 and mixed(1, t=0) == 5 and mixed(3, t=0) == 5 and mixed(0) == 1      # the last one: no scales of w
    assert L.htr_product_rounds(16, 1, 0) == 1 and L.htr_product_rounds(17, 1, 0) == 0 and L.htr_product_rounds(256, 64, 1) == 1 and L.htr_product_rounds(257, 64, 1) == 0
    need = L.htr_moe_stacked_scratch_bytes
    assert need(4, 2, 8, 256, 128, 3) > 0 and need(0, 2, 8, 256, 128, 3) == 0 and need(4, 2, 8, 256, 72, 3) == 0 and need(4, 2, 8, 256, 72, 0) > 0
    assert need(4, 2, 8, 256, 128, 2) == 0 and need(1 << 24, 4096, 8, 256, 128, 0) == 0
    a256 = ctypes.c_void_p(0x100000)
    moe = lambda x=p, dt=0, t=0, gus=None, sc=a256, bytes=1 << 30, y=p, T=4: \
        L.htr_moe_stacked(x, dt, p, 1, p, T, 2, p, gus, p, gus, 8, 256, 128, t, y, sc, bytes, None)
    assert moe(T=0) == 11 and moe(dt=2) == 5 and moe(dt=1) == 5 and moe(t=3) == 1 and moe(x=None) == 1 and moe(y=odd) == 7
    assert moe(sc=None) == 6 and moe(sc=ctypes.c_void_p(0x1010)) == 6 and moe(bytes=100) == 6


# ---- the C++ host path and the Python one
@pytest.mark.gpu
def test_both_host_paths_agree(gen, monkeypatch):
    x, w = randn(gen, 5, 256, dtype=BF16), randn(gen, 256, dtype=BF16)
    r, b = randn(gen, 5, 256, dtype=BF16), randn(gen, 64, dtype=BF16)
    q, s = fp8_weight(gen, 64, 256)
    gu8, dn8 = fp8_weight(gen, 3, 256, 256), fp8_weight(gen, 3, 256, 128)
    gu, dn = randn(gen, 3, 256, 256, dtype=BF16), randn(gen, 3, 256, 128, dtype=BF16)
    ends = torch.tensor([2, 2, 4], dtype=torch.int32, device="cuda")
    ids, wt = torch.tensor([[0, 2], [1, 1], [2, 0], [0, 1], [2, 2]], device="cuda"), torch.rand(5, 2, device="cuda", generator=gen)
    xq = ops.quantize_fp8(x)
    calls = [lambda: ops.rms_norm(x, w), lambda: ops.rms_norm(x, w, 1e-5, residual=r), lambda: ops.rms_norm(x, w, residual=r, quantize=True),
             lambda: ops.rms_norm(x, w, quantize=True), lambda: ops.linear_fp8(x, q, s, b), lambda: ops.linear_fp8(xq, q, s, out_dtype=F32),
             lambda: ops.linear_fp8(x.float(), q, s), lambda: ops.grouped_mm(x, gu, ends), lambda: ops.grouped_mm(xq, gu8, ends),
             lambda: ops.grouped_mm(x, gu8, ends, out_dtype=F16), lambda: ops.moe_experts_stacked(x, ids, wt, gu, dn),
             lambda: ops.moe_experts_stacked(x, ids, wt, gu8, dn8)]
    flat = lambda o: [o] if isinstance(o, torch.Tensor) else [t for p in o for t in flat(p)]
    taken = []
    fast = _native.fast()
    assert fast is not None

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
            assert u.dtype == v.dtype and u.shape == v.shape and torch.equal(u.float(), v.float())


@pytest.mark.gpu
def test_the_cxx_path_leaves_the_rest_to_python(gen):
    """What it does not take is handled by the other path, or refused there: it queues nothing and raises nothing."""
    fast, stream = _native.fast(), torch.cuda.current_stream().cuda_stream
    x, w = randn(gen, 4, 256, dtype=BF16), randn(gen, 256, dtype=BF16)
    q, s = fp8_weight(gen, 64, 256)
    for a in ((x[:, ::2], w[:128]), (x[:, 1:129], w[:128]), (x.double(), w.double()), (x, w[:255]), (x, w.float()), (x.cpu(), w), (x, w.cpu()), (x[:0], w), (3, w),
              (x, None), (x.clone().requires_grad_(), w)):
        assert fast.rms_norm(*a, 1e-6, None, False, stream) is None
    assert fast.rms_norm(x, w, 1e-6, x[:2], False, stream) is None and fast.rms_norm(x[:, :200].contiguous(), w[:200], 1e-6, None, True, stream) is None
    for a in ((x, None, q, s[:, :1], None, None, 0), (x, None, q.float(), s, None, None, 0), (x, None, q, s, w, None, 0), (x, None, q, s, None, None, 3),
              (x, None, q, s, None, None, -1), (x, s, q, s, None, None, 0), (x.double(), None, q, s, None, None, 0), (x, None, w, None, None, None, 0),
              (x, None, x[None], None, None, None, 0), (x, None, x[None], None, None, torch.ones(1, device="cuda"), 0), (x[:, 1:], None, q, s, None, None, 0),
              (x, None, q, s.cpu(), None, None, 0), (x, None, q.T, s, None, None, 0)):
        assert fast.product(*a, stream) is None
    ids, wt, gu, dn = torch.zeros(4, 1, dtype=torch.int64, device="cuda"), torch.ones(4, 1, device="cuda"), randn(gen, 1, 16, 256, dtype=BF16), randn(gen, 1, 256, 8, dtype=BF16)
    for a in ((x, ids.float(), wt, gu, None, dn, None), (x, ids, wt.double(), gu, None, dn, None), (x, ids[:2], wt, gu, None, dn, None), (x, ids, wt, gu, None, dn[:, :8], None),
              (x, ids, wt, gu, s, dn, None), (x.float(), ids, wt, gu, None, dn, None), (x, ids, wt, gu.half(), None, dn, None), (x, ids, wt, gu[:, :15], None, dn, None)):
        assert fast.moe_stacked(*a, stream) is None
    with pytest.raises(TypeError):
        fast.bind_unpacked(0)
