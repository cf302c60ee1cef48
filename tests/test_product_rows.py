"""The kernels that stream a matrix for few rows, in 16 bits and in int8, on rows that end with a slab of 128 bytes and on rows that end inside one: two instances of each kernel.

Each case names the kernel that it is for, and a test without a GPU holds it to that.  Tolerances as in test_product_kernels.py and test_int8.py."""
import pytest
import torch

import test_int8
from htr_amd import ops
from test_int8_tiles import plan as plan_int8
from test_product_kernels import BF16, F16, F32, assert_within, fenced, gen, plan, product_bound, randn, uneven  # noqa: F401

# experts (0: one matrix, no ends), rows, m, bytes of a row, then {matrix rows of a tile, rows of x, waves, stages}
IN_16_BITS = [
    (4, 9, 200, 640, (16, 16, 8, 0)), (4, 9, 200, 656, (16, 16, 8, 0)), (1, 1, 40, 128, (16, 16, 8, 0)), (1, 2, 40, 16, (16, 16, 8, 0)),
    (3, 12, 4100, 1408 * 2, (16, 16, 8, 0)), (3, 12, 4100, 1416 * 2, (16, 16, 8, 0)),
    (3, 5, 300, 8192, (16, 16, 16, 0)), (3, 5, 300, 8208, (16, 16, 16, 0)), (1, 4, 1030, 16384, (16, 16, 16, 0)), (1, 3, 1030, 16272, (16, 16, 16, 0)),
    (2, 4, 9001, 256, (32, 16, 4, 0)), (2, 4, 9001, 144, (32, 16, 4, 0)),
    (2, 40, 1542, 2048, (16, 32, 8, 0)), (2, 40, 1542, 2064, (16, 32, 8, 0)), (4, 60, 1024, 4096, (16, 32, 8, 0)), (4, 60, 1024, 4112, (16, 32, 8, 0)),
    (2, 40, 1542, 112, (16, 32, 8, 0)),
]
IN_INT8 = [
    (0, 33, 1542, 1024, (16, 32, 8, 0)), (0, 33, 1542, 1040, (16, 32, 8, 0)), (0, 60, 200, 112, (16, 16, 8, 0)), (0, 60, 200, 128, (16, 16, 8, 0)),
    (8, 80, 512, 4096, (16, 32, 8, 0)), (8, 80, 512, 4112, (16, 32, 8, 0)),
    (0, 3, 300, 98304, (16, 16, 16, 0)), (0, 3, 300, 98320, (16, 16, 16, 0)), (0, 3, 5000, 65536, (16, 16, 8, 0)), (0, 3, 5000, 65552, (16, 16, 8, 0)),
    (8, 48, 72, 24592, (16, 16, 8, 0)), (8, 48, 72, 24576, (16, 16, 8, 0)),
]


def test_every_kernel_has_both_kinds_of_rows():
    for cases, kernels, of in ((IN_16_BITS, {(16, 16, 8, 0), (16, 16, 16, 0), (32, 16, 4, 0), (16, 32, 8, 0)}, lambda E, rows, m, b: plan(rows, m, b // 2, E, True, False, BF16)),
                               (IN_INT8, {(16, 16, 8, 0), (16, 16, 16, 0), (16, 32, 8, 0)}, lambda E, rows, m, b: plan_int8(rows, m, b, max(E, 1), E > 0))):
        seen = set()
        for E, rows, m, b, kernel in cases:
            assert of(E, rows, m, b)[:4] == kernel, (E, rows, m, b, of(E, rows, m, b))
            seen.add((kernel, b % 128 != 0))
        assert seen == {(k, tail) for k in kernels for tail in (False, True)}


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [BF16, F16])
@pytest.mark.parametrize("case", IN_16_BITS, ids=lambda c: "x".join(map(str, c[:4])))
def test_in_16_bits(gen, kind, case):
    E, rows, m, b = case[:4]
    n, counts = b // 2, uneven(E, rows)
    ends = torch.tensor(counts, dtype=torch.int32).cumsum(0).to(torch.int32).cuda()
    w, x = fenced(randn(gen, E, m, n, dtype=kind, scale=n ** -0.5)), fenced(randn(gen, rows, n, dtype=kind))
    y = ops.grouped_mm(x, w, ends, out_dtype=F32)
    first = 0
    for e, c in enumerate(counts):
        if c:
            assert_within(y[first:first + c], *product_bound(x[first:first + c], w[e], F32))
        first += c


@pytest.mark.gpu
@pytest.mark.parametrize("case", IN_INT8, ids=lambda c: "x".join(map(str, c[:4])))
def test_in_int8(gen, case):
    E, rows, m, n = case[:4]
    x, w = tuple(map(fenced, ops.quantize_int8(randn(gen, rows, n)))), tuple(map(fenced, test_int8.weight(gen, max(E, 1), m, n)))
    if E:
        counts = uneven(E, rows)
        test_int8.check_grouped(x, w, counts, F32, ops.grouped_mm(x, w, test_int8._ends(counts), out_dtype=F32))
    else:
        test_int8.assert_within(ops.linear_int8(x, w[0][0], w[1][0], out_dtype=F32), *test_int8.product_bound(x, (w[0][0], w[1][0]), F32))
