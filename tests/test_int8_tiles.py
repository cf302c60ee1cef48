"""The int8 tiles for many rows by the plan that the library says it takes, against 64 bits: grouped products, and gate and up of a routed layer in one launch.

Each case names the kernel that it is for, and a test without a GPU holds it to that.  Every kernel has rows of as many slabs of 128 bytes as its ring has stages, where the next
tile's scales are asked for as the tile's first slab is multiplied, and of one more; with and without a last slab that ends early; each with more tiles than workgroups, so that
the two places for a tile's scales turn.  Sums are exact; what follows is bounded as in test_int8.py."""
import ctypes

import pytest
import torch

from htr_amd import _native, ops
from test_int8 import BF16, F16, F32, I8, _ends, assert_within, check_grouped, experts, gen, half_step, moe64, product, randn, rounded, value, weight  # noqa: F401
from test_product_kernels import GATED, RING, fenced, ids, uneven


def plan(rows, m, n, experts=1, grouped=True, gated=False):
    """(matrix rows of a tile, rows of x, waves, stages, workgroups, tiles) or the status."""
    out = (ctypes.c_int * 6)()
    rc = _native.lib().htr_product_plan(rows, m, n, experts, int(grouped), int(gated), _native.I8, _native.I8, out)
    return tuple(out) if rc == 0 else rc


GROUPED_CASES = [      # experts, rows, m, n, {matrix rows, rows of x, waves, stages}, several tiles to a workgroup
    (66, 1599, 1000, 432, (64, 32, 4, 4), True),
    (22, 543, 3000, 560, (64, 32, 4, 4), True),
    (30, 1170, 920, 432, (64, 64, 4, 4), True),
    (20, 780, 1440, 640, (64, 64, 4, 4), True),
    (66, 594, 523, 512, (128, 32, 4, 4), True),
    (22, 198, 2080, 560, (128, 32, 4, 4), True),
    (22, 543, 4104, 304, (128, 64, 4, 3), True),
    (66, 4290, 523, 512, (128, 64, 4, 3), True),
    (66, 7920, 523, 384, (128, 128, 4, 3), True),
    (16, 11200, 523, 432, (128, 128, 4, 3), True),
    (22, 1430, 4104, 304, (256, 128, 8, 3), True),
    (66, 5940, 1032, 432, (256, 128, 8, 3), True),
    (22, 4400, 4104, 256, (256, 256, 8, 2), True),
    (66, 17160, 1032, 304, (256, 256, 8, 2), True),
]
GATED_CASES = [      # experts, rows, 2 F, H
    (1, 10, 32, 512, (256, 32, 4, 4), False),
    (5, 46, 32, 560, (256, 32, 4, 4), False),
    (66, 596, 1568, 432, (256, 32, 4, 4), True),
    (16, 146, 6176, 640, (256, 32, 4, 4), True),
    (16, 8320, 32, 304, (256, 64, 4, 3), False),
    (66, 1332, 1568, 384, (256, 64, 4, 3), True),
    (24, 592, 4128, 432, (256, 64, 4, 3), True),
    (24, 16800, 32, 432, (256, 128, 8, 3), False),
    (66, 2606, 1568, 304, (256, 128, 8, 3), True),
    (16, 800, 6176, 512, (256, 128, 8, 3), True),
    (24, 16800, 288, 256, (256, 256, 8, 2), False),
    (66, 46200, 288, 256, (256, 256, 8, 2), True),
    (24, 6240, 3104, 304, (256, 256, 8, 2), True),
]


def test_every_tile_has_its_cases():
    for gated, cases, kernels in ((False, GROUPED_CASES, RING), (True, GATED_CASES, GATED)):
        turned = set()
        for E, rows, m, n, kernel, several in cases:
            p = plan(rows, m, n, E, True, gated)
            assert p[:4] == kernel, (E, rows, m, n, p)
            tiles = -(-m // kernel[0]) * sum(-(-c // kernel[1]) for c in uneven(E, rows))
            assert tiles <= p[5] and (tiles > p[4]) == several, (tiles, p)
            if several:
                turned.add((kernel, -(-n // 128) - kernel[3]))
        assert turned == {(k, more) for k in kernels for more in (0, 1)}
        assert {n % 128 != 0 for _, _, _, n, _, _ in cases} == {True, False}


# ---- grouped products
@pytest.mark.gpu
@pytest.mark.parametrize("case", GROUPED_CASES, ids=ids(GROUPED_CASES))
def test_grouped(gen, case):
    E, rows, m, n, kernel, several = case
    counts, behind = uneven(E, rows), 37
    if plan(rows + behind, m, n, E)[:4] != kernel:
        behind = 0
    x = tuple(map(fenced, ops.quantize_int8(randn(gen, rows + behind, n) * torch.exp(randn(gen, rows + behind, 1)))))
    w = tuple(map(fenced, weight(gen, E, m, n)))
    for dtype in (BF16, F32):
        y = ops.grouped_mm(x, w, _ends(counts), out_dtype=dtype)
        check_grouped(x, w, counts, dtype, y)
    assert torch.equal(ops.grouped_mm(x, w, _ends(counts), out_dtype=F32), y)


# ---- routed layers
def layer64(x, ids, wt, gate_up, down, dtype):
    """test_int8's moe64, an expert's pairs at once."""
    (T, H), top = x.shape, ids.shape[1]
    q = rounded(x.double())
    y, bound = torch.zeros(T, H, dtype=torch.float64, device=x.device), torch.zeros(T, H, dtype=torch.float64, device=x.device)
    flat, p = ids.reshape(-1), wt.reshape(-1).double()
    for e in range(gate_up[0].shape[0]):
        pairs = torch.nonzero(flat == e)[:, 0]
        if not len(pairs):
            continue
        tok, pe = pairs // top, p[pairs][:, None]
        g, u = product((q[0][tok], q[1][tok]), (gate_up[0][e], gate_up[1][e])).chunk(2, -1)
        h = g * torch.sigmoid(g) * u
        off = h.abs() * 2.0 ** -20 * (1 + g.abs())
        hq, s = rounded(h)
        z = (h / s[:, None]).abs()
        moved = (off.amax(-1) / h.abs().amax(-1).clamp(min=2.0 ** -100) + 2.0 ** -23)[:, None]
        flips = (((z - torch.floor(z)) - 0.5).abs() <= off / s[:, None] + z * moved).double()
        wd = value(down[0][e], down[1][e]).abs().T
        out = product((hq, s), (down[0][e], down[1][e]))
        part = ((flips @ wd) * s[:, None] + ((hq * s[:, None]).abs() @ wd) * moved + out.abs() * 2.0 ** -22) * (1 + 2.0 ** -22)
        y.index_add_(0, tok, pe * out)
        bound.index_add_(0, tok, pe.abs() * part + (pe * out).abs() * 2.0 ** -23)
    y[((ids < 0) | (ids >= gate_up[0].shape[0])).any(-1)] = float("nan")
    bound += (bound + y.abs()).nan_to_num(0.0) * top * 2.0 ** -23
    return y, bound * 1.01 + half_step(y.abs() + bound, dtype)


def test_the_definition_by_expert_is_the_one_by_token():
    gen = torch.Generator().manual_seed(20261209)
    T, E, top, H, F = 13, 5, 3, 64, 48
    gate_up, down = experts(gen, E, H, F)
    x, wt, ids = randn(gen, T, H, dtype=BF16), torch.rand(T, top, generator=gen), torch.randint(0, E, (T, top), generator=gen)
    ids[4, 1] = -1
    a, b = layer64(x, ids, wt, gate_up, down, BF16), moe64(x, ids, wt, gate_up, down, BF16)
    for u, v in zip(a, b):
        assert torch.allclose(u, v, rtol=1e-9, atol=1e-12, equal_nan=True)


def layer(gen, T, top, E, H, F, dtype, counts):
    """Inputs of a layer whose experts have exactly these rows."""
    flat = torch.repeat_interleave(torch.arange(E), torch.tensor(counts))
    flat = flat[torch.randperm(T * top, generator=torch.Generator().manual_seed(7))]
    gate_up, down = (tuple(map(fenced, w)) for w in experts(gen, E, H, F))
    return fenced(randn(gen, T, H, dtype=dtype)), flat.view(T, top).cuda(), torch.rand(T, top, device="cuda", generator=gen), gate_up, down


@pytest.mark.gpu
@pytest.mark.parametrize("case", GATED_CASES, ids=ids(GATED_CASES))
def test_gated(gen, case):
    E, rows, m, n, kernel, several = case
    dtype = F16 if E % 2 else BF16
    call = layer(gen, rows // 2, 2, E, n, m // 2, dtype, uneven(E, rows))
    y = ops.moe_experts_stacked(*call)
    assert_within(y, *layer64(*call, dtype))
    assert torch.equal(ops.moe_experts_stacked(*call), y)
    call[0][3, n // 2] = float("nan")
    z = ops.moe_experts_stacked(*call)
    assert z[3].isnan().all()
    z[3] = y[3]
    assert torch.equal(z, y)


# a layer and a linear whose launches all have several tiles to a workgroup
T, TOP, E, H, F, M = 3000, 4, 16, 1040, 1040, 6000


def test_all_launches_of_the_streams_test_go_on_from_tile_to_tile():
    counts = uneven(E, T * TOP)
    for rows, m, n, gated, of in ((T * TOP, 2 * F, H, True, counts), (T * TOP, H, F, False, counts), (T, M, H, None, [T])):
        p = plan(rows, m, n, 1 if gated is None else E, gated is not None, bool(gated))
        assert -(-m // p[0]) * sum(-(-c // p[1]) for c in of) > p[4], (rows, m, n, p)


@pytest.mark.gpu
def test_tiles_that_go_on_on_two_streams_and_replayed(gen):
    call, w = layer(gen, T, TOP, E, H, F, BF16, uneven(E, T * TOP)), weight(gen, M, H)
    y = ops.moe_experts_stacked(*call)
    assert_within(y, *layer64(*call, BF16))
    run = lambda x: ops.linear_int8(ops.moe_experts_stacked(x, *call[1:]), *w)
    inputs = [call[0]] + [randn(gen, T, H, dtype=BF16) for _ in range(3)]
    want = [run(x) for x in inputs]
    pair = ops.quantize_int8(y)
    exact = product(pair, w)
    assert_within(want[0], exact, exact.abs() * 3.01 * 1.01 * 2.0 ** -24 + half_step(exact.abs() * (1 + 2.0 ** -22), BF16))
    side, got = [torch.cuda.Stream() for _ in range(2)], []
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
