"""ops.route_experts against its definition, token by token in 64 bits on the CPU.

Weights: scores and sums in 64 bits, rounded once to float32: off by half a step, 2^-24 relative (and 64-bit roundings, 2^-40 here for all of them)."""
import ctypes
import math

import pytest
import torch

from htr_amd import _native, ops

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture
def gen():
    return torch.Generator(device="cuda").manual_seed(20261208)


def route64(logits, top, scores="softmax", bias=None, groups=1, top_groups=1, group_best=1, renormalize=True, scale=1.0):
    """One token at a time; NaN counts as more than anything."""
    bias = None if bias is None else bias.double().cpu().tolist()
    all_ids, all_weights = [], []
    for l in logits.double().cpu().reshape(-1, logits.shape[-1]):
        s = torch.softmax(l, -1) if scores == "softmax" else torch.sigmoid(l)
        if (l == -math.inf).all():
            s = torch.zeros_like(l)
        l, s = l.tolist(), s.tolist()
        masked = [v == -math.inf or (bias is not None and bias[e] == -math.inf) for e, v in enumerate(l)]
        with_bias = [v + (0.0 if bias is None else bias[e]) for e, v in enumerate(s)]
        rank = [-math.inf if masked[e] else with_bias[e] if bias is not None else l[e] for e in range(len(l))]
        by_group = with_bias if group_best == 2 else rank
        by_group = [-math.inf if masked[e] else by_group[e] for e in range(len(l))]
        key = lambda v: (0, 0.0) if math.isnan(v) else (1, -v)
        size = len(l) // groups
        best = [sum(sorted(by_group[g * size:(g + 1) * size], key=key)[:group_best]) for g in range(groups)]
        inside = sorted(range(groups), key=lambda g: (key(best[g]), g))[:top_groups]
        rank = [v if groups == 1 or e // size in inside else -math.inf for e, v in enumerate(rank)]
        ids = sorted(range(len(l)), key=lambda e: (key(rank[e]), e))[:top]
        w = [0.0 if rank[e] == -math.inf else s[e] for e in ids]
        total = sum(w)
        if renormalize:
            w = [v / total if total != 0 else 0.0 for v in w]
        all_ids.append(ids)
        all_weights.append([v * scale for v in w])
    shape = logits.shape[:-1] + (top,)
    return torch.tensor(all_ids, dtype=torch.int32).reshape(shape), torch.tensor(all_weights, dtype=torch.float64).reshape(shape)


def check(logits, top, **how):
    ids, weights = ops.route_experts(logits, top, **how)
    want, exact = route64(logits, top, **how)
    assert ids.dtype == torch.int32 and weights.dtype == F32 and ids.shape == weights.shape == want.shape
    assert torch.equal(ids.cpu(), want)
    w = weights.double().cpu()
    assert torch.equal(w.isnan(), exact.isnan())
    off = (w - exact).abs().nan_to_num(0.0) - exact.abs().nan_to_num(0.0) * (2.0 ** -24 + 2.0 ** -40) - 2.0 ** -149
    assert off.max().item() <= 0 if off.numel() else True
    return ids, weights


def randn(gen, *shape, dtype=F32, scale=1.0):
    return (torch.randn(*shape, device=gen.device, generator=gen) * scale).to(dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
@pytest.mark.parametrize("with_bias", [False, True])
@pytest.mark.parametrize("E,top", [(1, 1), (2, 2), (7, 3), (60, 4), (64, 6), (65, 8), (128, 8), (160, 6), (256, 8), (257, 1), (384, 8), (512, 10), (777, 64), (1024, 32)])
def test_route(gen, dtype, scores, with_bias, E, top):
    for tokens, renormalize, scale in ((1, True, 1.0), (33, False, 2.5), (70, True, 0.5)):
        logits = randn(gen, tokens, E, dtype=dtype, scale=2)
        bias = randn(gen, E, scale=0.1) if with_bias else None
        check(logits, top, scores=scores, bias=bias, renormalize=renormalize, scale=scale)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("scores,with_bias", [("softmax", False), ("sigmoid", True), ("sigmoid", False), ("softmax", True)])
@pytest.mark.parametrize("E,groups,top_groups,top", [(8, 2, 1, 4), (64, 8, 4, 8), (60, 4, 2, 5), (256, 8, 4, 8), (160, 8, 3, 6), (96, 3, 1, 20), (64, 64, 5, 5), (512, 16, 1, 32),
                                                     (1024, 64, 7, 64), (72, 8, 8, 3), (256, 1, 1, 8), (320, 5, 2, 9)])
@pytest.mark.parametrize("group_best", [1, 2])
def test_route_in_groups(gen, dtype, scores, with_bias, E, groups, top_groups, top, group_best):
    logits = randn(gen, 41, E, dtype=dtype, scale=2)
    bias = randn(gen, E, scale=0.1) if with_bias else None
    check(logits, top, scores=scores, bias=bias, groups=groups, top_groups=top_groups, group_best=group_best)


@pytest.mark.gpu
@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
@pytest.mark.parametrize("E,groups,top_groups", [(64, 1, 1), (256, 8, 4), (24, 4, 2)])
def test_ties_go_to_the_lowest_number(gen, scores, E, groups, top_groups):
    for values in (1, 2, 5):
        logits = torch.randint(0, values, (50, E), device="cuda", generator=gen).to(BF16)
        logits[0] = 0
        logits[1, ::2] = -0.0
        logits[2] = 60        # sigmoids of 1
        for bias in (None, torch.zeros(E, device="cuda"), torch.randint(0, 2, (E,), device="cuda", generator=gen).float() / 4):
            for group_best in (1, 2):
                check(logits, 7, scores=scores, bias=bias, groups=groups, top_groups=top_groups, group_best=group_best)


@pytest.mark.gpu
@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
@pytest.mark.parametrize("E,groups,top_groups", [(64, 1, 1), (256, 8, 4), (24, 4, 2)])
def test_masked_experts_infinities_and_nan(gen, scores, E, groups, top_groups):
    logits = randn(gen, 40, E)
    logits[0] = -math.inf                                     # nothing left
    logits[1, 3:] = -math.inf                                 # fewer left than are asked for
    logits[2, :E - 1] = -math.inf
    logits[3, ::3] = -math.inf
    logits[4, 5], logits[5, 2], logits[6, E - 1] = math.inf, math.nan, math.nan
    logits[7] = math.nan
    logits[8] = torch.finfo(F32).min                          # the type's lowest value masks nothing by itself
    logits[9, ::2] = torch.finfo(F32).min
    logits[10] = 1e30
    logits[11] = -1e30
    logits[12, : E // 2] = -math.inf
    masking = torch.where(torch.arange(E, device="cuda") % 5 == 2, -math.inf, randn(gen, E, scale=0.1))
    for bias in (None, randn(gen, E, scale=0.1), masking):
        for group_best in (1, 2):
            for renormalize in (True, False):
                check(logits, 6, scores=scores, bias=bias, groups=groups, top_groups=top_groups, group_best=group_best, renormalize=renormalize)
                check(logits[:1], 6, scores=scores, bias=bias, groups=groups, top_groups=top_groups, group_best=group_best, renormalize=renormalize)


@pytest.mark.gpu
def test_experts_whose_ranks_are_next_to_each_other(gen):
    """Differences that 64 bits hold and 32 do not."""
    E = 64
    logits = torch.zeros(200, E, device="cuda")
    bias = torch.zeros(E, device="cuda")
    bias[:] = 0.25
    step = 2.0 ** -26 * torch.arange(E, device="cuda")        # below a step of float32 at 3/4
    logits[:] = 4 * step[torch.argsort(torch.rand(200, E, device="cuda", generator=gen), -1)]       # sigmoid(x) = 1/2 + x / 4
    check(logits, 8, scores="sigmoid", bias=bias)
    check(logits, 8, scores="sigmoid", bias=bias, groups=8, top_groups=3, group_best=2)
    check(logits, 8, scores="softmax", bias=bias)


@pytest.mark.gpu
def test_route_takes_strides_any_alignment_and_leading_dimensions(gen):
    big = randn(gen, 6, 5, 201, dtype=BF16)
    for x in (big[:, 1, 3:67], big[::2, :, 1:101], big.transpose(1, 2)[:, :64, :], big[..., :150:2], big[0, 0, :7]):
        check(x, min(6, x.shape[-1]), scores="sigmoid", bias=randn(gen, x.shape[-1] + 1, dtype=BF16)[1:])
    wide = randn(gen, 70, 257)[:, 1:]
    check(wide, 8, scores="sigmoid", groups=8, top_groups=4, group_best=2)
    assert [t.shape for t in ops.route_experts(big[:0], 3)] == [(0, 5, 3)] * 2
    row = randn(gen, 64)
    check(row.expand(9, 64), 6)                               # rows of stride 0


@pytest.mark.gpu
def test_many_tokens(gen):
    logits, bias = randn(gen, 20000, 256, scale=1.5), randn(gen, 256, scale=0.05)
    how = dict(scores="sigmoid", bias=bias, groups=8, top_groups=4, group_best=2, scale=2.5)
    ids, weights = ops.route_experts(logits, 8, **how)
    for first in (0, 9999, 19950):
        a, b = ops.route_experts(logits[first:first + 50].clone(), 8, **how)
        assert torch.equal(ids[first:first + 50], a) and torch.equal(weights[first:first + 50], b)
    check(logits[:300], 8, **how)
    for tokens in (5, 17, 100, 1000):                         # a token's result does not depend on how many come with it
        a, b = ops.route_experts(logits[:tokens], 8, **how)
        assert torch.equal(ids[:tokens], a) and torch.equal(weights[:tokens], b)


@pytest.mark.gpu
def test_more_tokens_than_a_launch_takes(gen):
    tokens = (1 << 22) + 5
    logits = randn(gen, tokens, 8, dtype=BF16)
    ids, weights = ops.route_experts(logits, 2)
    a, b = ops.route_experts(logits[-9:].clone(), 2)
    assert torch.equal(ids[-9:], a) and torch.equal(weights[-9:], b)


@pytest.mark.gpu
def test_router_and_experts_on_streams_and_captured(gen):
    """As they are used: a router in front of the routed layer, eager on two streams at once, and replayed."""
    H, F, E = 256, 128, 16
    gu, dn = ops.quantize_weight_int8(randn(gen, E, 2 * F, H, scale=H ** -0.5)), ops.quantize_weight_int8(randn(gen, E, H, F, scale=F ** -0.5))
    router, bias = randn(gen, E, H, scale=H ** -0.5), randn(gen, E, scale=0.1)

    def run(x):
        ids, p = ops.route_experts(x.float() @ router.T, 3, scores="sigmoid", bias=bias, groups=4, top_groups=2, group_best=2, scale=1.5)
        return ops.moe_experts_stacked(x, ids, p, gu, dn)

    inputs = [randn(gen, 11, H, dtype=BF16) for _ in range(4)]
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
        run(inputs[(k + 1) % 4])                              # eager work between the replays
        torch.cuda.synchronize()
        assert torch.equal(out, want[k])
    for a, b in zip(torch.compile(lambda x: ops.route_experts(x, 2), backend="eager")(inputs[0]), ops.route_experts(inputs[0], 2)):
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_router_in_front_of_packed_experts(gen):
    from htr_amd import wire
    E, H, F, T = 4, 256, 128, 5
    matrices = lambda m, n, seed: [tuple(t.cuda() for t in wire.synth_linear(m, n, 4, seed + e)) for e in range(E)]
    gu, dn = matrices(2 * F, H, 100), matrices(H, F, 200)
    x, logits = randn(gen, T, H, dtype=BF16), randn(gen, T, E)
    logits[2] = -math.inf                                     # a padded token: weights 0
    ids, weights = ops.route_experts(logits, 2)
    y = ops.moe_experts(x, ids, weights, gu, dn)
    assert torch.equal(y, ops.moe_experts(x, ids.long(), weights, gu, dn)) and (y[2] == 0).all() and y.isfinite().all() and (y[0] != 0).any()


# ---- refusals
def wrong_calls(device):
    x = torch.zeros(2, 64, device=device)
    route = ops.route_experts
    return [lambda: route(x, 0), lambda: route(x, 65), lambda: route(torch.zeros(2, 128, device=device), 65), lambda: route(x.double(), 2), lambda: route(x[0, 0], 1),
            lambda: route(x[:, :0], 1), lambda: route(torch.zeros(1, 1025, device=device), 1), lambda: route(x, 2, scores="exp"), lambda: route(x, 2, scores=None),
            lambda: route(x, 2, groups=5), lambda: route(x, 2, groups=0), lambda: route(x, 2, groups=8, top_groups=9), lambda: route(x, 2, groups=8, top_groups=0),
            lambda: route(x, 9, groups=8, top_groups=1), lambda: route(x, 2, groups=8, group_best=3), lambda: route(x, 2, bias=x), lambda: route(x, 2, bias=x[0, :63]),
            lambda: route(x, 2, bias=x[0].double()), lambda: route(torch.zeros(2, 128, device=device), 2, groups=128), lambda: route(x, -1)]


def test_refusals_without_a_gpu():
    with pytest.raises(RuntimeError, match="ROCm device only"):
        ops.route_experts(torch.zeros(2, 64), 2)
    for k, call in enumerate(wrong_calls("cpu")):
        with pytest.raises(RuntimeError, match="route_experts"):
            call()
            pytest.fail(f"call {k} was taken")


@pytest.mark.gpu
def test_refusals_on_a_gpu(gen):
    for k, call in enumerate(wrong_calls("cuda")):
        with pytest.raises(RuntimeError, match="route_experts"):
            call()
            pytest.fail(f"call {k} was taken")
    x, b = randn(gen, 2, 64), randn(gen, 64)
    with pytest.raises(RuntimeError, match="device of x"):
        ops.route_experts(x, 2, bias=b.cpu())
    for call in (lambda: ops.route_experts(x.clone().requires_grad_(), 2), lambda: ops.route_experts(x, 2, bias=b.clone().requires_grad_())):
        with pytest.raises(RuntimeError, match="no derivative"):
            call()
        with torch.no_grad():
            call()


def test_status_codes_without_a_gpu():
    L = _native.lib()
    p, odd = ctypes.c_void_p(0x1000), ctypes.c_void_p(0x1001)          # never dereferenced: every call is refused first, or does nothing
    route = lambda x=p, dt=2, T=1, E=64, top=2, b=None, groups=1, tg=1, gb=1, ids=p, w=p: L.htr_route(x, E, dt, T, E, top, 0, b, groups, tg, gb, 1, 1.0, ids, w, None)
    assert route(T=0) == 0 and route(T=-1) == 11 and route(E=0) == 11 and route(E=1025) == 11 and route(top=0) == 11 and route(top=65) == 11 and route(dt=3) == 5
    assert route(groups=3) == 11 and route(groups=4, tg=5) == 11 and route(groups=32, tg=1, top=3) == 11 and route(groups=4, gb=3) == 11 and route(E=128, groups=128) == 11
    assert route(x=None) == 1 and route(ids=None) == 1 and route(w=None) == 1 and route(x=odd) == 7 and route(b=odd) == 7 and route(ids=odd) == 7 and route(w=odd) == 7


@pytest.mark.gpu
def test_both_host_paths_agree(gen, monkeypatch):
    x, bias = randn(gen, 3, 7, 64, dtype=BF16), randn(gen, 64)
    calls = [lambda: ops.route_experts(x, 6), lambda: ops.route_experts(x, 6, scores="sigmoid", bias=bias, groups=8, top_groups=2, group_best=2, renormalize=False, scale=3.0)]
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
        got = call()
        assert taken == [("route", True)]
        monkeypatch.setattr(_native, "fast", lambda: None)
        assert all(torch.equal(a, b) and a.dtype == b.dtype and a.shape == b.shape for a, b in zip(got, call()))
