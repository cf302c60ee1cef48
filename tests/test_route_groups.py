"""ops.route_experts on groups of experts, some of them masked, against what its documentation says, expert by expert in 64 bits on the CPU.

A masked expert (logit or bias of -inf) has no part in anything: a group is as good as the sum of its up to group_best best experts that are not masked, and one without any is
behind all others.  Weights are 64 bits rounded once to float32: off by half a step, 2^-24 relative (and 64-bit roundings, 2^-40 here for all of them)."""
import math

import pytest
import torch

from htr_amd import ops

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture
def gen():
    return torch.Generator(device="cuda").manual_seed(20261209)


def routed(l, top, scores, bias, groups, top_groups, group_best, renormalize, scale):
    """(ids, weights) of one token's logits, a list of Python floats."""
    E, size = len(l), len(l) // groups
    if scores == "sigmoid":
        s = [v if math.isnan(v) else 1 / (1 + math.exp(-v)) if v >= 0 else math.exp(v) / (1 + math.exp(v)) for v in l]
    else:
        s = torch.softmax(torch.tensor(l, dtype=torch.float64), 0).tolist() if any(v != -math.inf for v in l) else [0.0] * E
    live = [l[e] != -math.inf and (bias is None or bias[e] != -math.inf) for e in range(E)]
    ranks = [l[e] if bias is None else s[e] + bias[e] for e in range(E)]
    best_first = lambda of: lambda e: (not math.isnan(of[e]), -of[e] if not math.isnan(of[e]) else 0.0, e)
    inside = range(groups)
    if groups > 1:
        values = ranks if bias is not None or group_best == 1 else s
        merit = []
        for g in range(groups):
            left = sorted((e for e in range(g * size, (g + 1) * size) if live[e]), key=best_first(values))[:group_best]
            merit.append(sum(values[e] for e in left) if left else -math.inf)
        inside = sorted(inside, key=best_first(merit))[:top_groups]
    competing = sorted((e for e in range(E) if live[e] and e // size in inside), key=best_first(ranks))[:top]
    others = sorted(e for e in range(E) if not (live[e] and e // size in inside))
    ids = (competing + others)[:top]
    w = [s[e] for e in competing] + [0.0] * (top - len(competing))
    if renormalize:
        total = sum(w)
        w = [v / total if total != 0 else 0.0 for v in w]
    return ids, [v * scale for v in w]


def check(logits, top, scores="softmax", bias=None, groups=1, top_groups=1, group_best=1, renormalize=True, scale=1.0):
    how = dict(scores=scores, groups=groups, top_groups=top_groups, group_best=group_best, renormalize=renormalize, scale=scale)
    ids, weights = ops.route_experts(logits, top, bias=bias, **how)
    b = None if bias is None else bias.double().cpu().tolist()
    want = [routed(l, top, bias=b, **how) for l in logits.double().cpu().tolist()]
    assert ids.cpu().tolist() == [w[0] for w in want]
    exact, w = torch.tensor([w[1] for w in want], dtype=torch.float64), weights.double().cpu()
    assert torch.equal(w.isnan(), exact.isnan())
    off = (w - exact).abs().nan_to_num(0.0) - exact.abs().nan_to_num(0.0) * (2.0 ** -24 + 2.0 ** -40) - 2.0 ** -149
    assert off.max().item() <= 0
    return ids, weights


def randn(gen, *shape, dtype=F32, scale=1.0):
    return (torch.randn(*shape, device=gen.device, generator=gen) * scale).to(dtype)


def test_the_definition_without_a_gpu():
    """By hand: one expert left, in the last group."""
    l = [-math.inf] * 7 + [2.0]
    for scores in ("softmax", "sigmoid"):
        for best in (1, 2):
            for bias in (None, [-3.0] * 8):
                ids, w = routed(l, 3, scores, bias, 4, 2, best, True, 1.0)
                assert ids == [7, 0, 1] and w == [1.0, 0.0, 0.0]
    assert routed([-math.inf] * 8, 2, "sigmoid", None, 4, 2, 2, True, 1.0) == ([0, 1], [0.0, 0.0])
    # 0.5 alone is less than 0.4 and 0.2, but with a bias of -0.35 more than 0.05 and -0.15
    l = [math.log(s / (1 - s)) for s in (0.4, 0.2, 0.5)] + [-math.inf]
    assert routed(l, 1, "sigmoid", None, 2, 1, 2, True, 1.0)[0] == [0]
    assert routed(l, 1, "sigmoid", [-0.35] * 4, 2, 1, 2, True, 1.0)[0] == [2]


KINDS = [("softmax", False), ("sigmoid", False), ("sigmoid", True), ("softmax", True)]


@pytest.mark.gpu
@pytest.mark.parametrize("scores,with_bias", KINDS)
@pytest.mark.parametrize("E,groups,top_groups,dtype", [(256, 8, 4, F32), (24, 4, 2, BF16), (64, 8, 1, F16), (60, 20, 3, F32), (256, 2, 1, BF16), (1023, 33, 2, F32), (64, 64, 3, F32),
                                                       (1005, 3, 1, F16)])
@pytest.mark.parametrize("group_best", [1, 2])
def test_groups_of_which_one_expert_is_left(gen, E, groups, top_groups, dtype, scores, with_bias, group_best):
    size, top, T = E // groups, min(6, E // groups * top_groups), 24
    logits = randn(gen, T, E, dtype=dtype)
    left = torch.zeros(T, E, dtype=torch.bool, device="cuda")
    left[0, E - 1] = True                                          # one, in the last group
    left[1, E // 2] = left[1, E - 1] = True                        # two, in different groups
    left[2, size - 1::size] = True                                 # one in each group
    left[3, E - size:] = True                                      # a group
    left[4, size // 2::size], left[4, :size] = True, True          # one in each but the first, which has all
    left[5:17] = torch.rand(12, E, device="cuda", generator=gen) < 2.0 / size
    left[17:T - 1] = torch.rand(T - 18, E, device="cuda", generator=gen) < 0.5
    logits[~left] = -math.inf                                      # the last token has none left
    how = dict(scores=scores, groups=groups, top_groups=top_groups, group_best=group_best)
    for bias in ((randn(gen, E, scale=0.3) - 1, torch.where(torch.arange(E, device="cuda") % 3 == 1, -math.inf, randn(gen, E, scale=0.1))) if with_bias else (None,)):
        for renormalize in (True, False):
            ids, weights = check(logits, top, bias=bias, renormalize=renormalize, **how)
            assert (weights[T - 1] == 0).all()
    # the same where 64 bits decide throughout: a bias beyond 2^60 of an expert that no token has left
    if with_bias:
        bias[0], logits[:, 0] = 2.0 ** 61, -math.inf
        check(logits, top, bias=bias, **how)
    logits[::2, E - 1] = math.nan
    check(logits, top, bias=bias, **how)


@pytest.mark.gpu
@pytest.mark.parametrize("scores,with_bias", KINDS)
@pytest.mark.parametrize("E,groups,top_groups,top", [(1023, 3, 2, 12), (1020, 5, 3, 8), (990, 33, 9, 8), (1023, 33, 4, 64), (1022, 2, 1, 64), (256, 2, 1, 8), (512, 2, 1, 17), (512, 2, 2, 8),
                                                     (260, 2, 1, 5), (1000, 5, 1, 33), (70, 35, 8, 10)])
@pytest.mark.parametrize("group_best", [1, 2])
def test_groups_of_many_lanes_and_of_one(gen, E, groups, top_groups, top, scores, with_bias, group_best):
    """Up to 31 experts to a lane; groups of 32 lanes, of 16 and of one; ranks next to each other, where 64 bits decide."""
    bias = randn(gen, E, scale=0.1) if with_bias else None
    how = dict(scores=scores, bias=bias, groups=groups, top_groups=top_groups, group_best=group_best)
    for logits in (randn(gen, 9, E, scale=2), randn(gen, 5, E, dtype=BF16), torch.randint(0, 4, (5, E), device="cuda", generator=gen).to(F16)):
        check(logits, top, **how)
    logits[1, 7] = math.inf
    check(logits, top, **how)
    # sigmoid(x) = 1/2 + x / 4 and a bias of 1/4: a quarter of float32's step at 3/4 from one to the next
    near = 2.0 ** -24 * torch.argsort(torch.rand(6, E, device="cuda", generator=gen), -1)
    check(near, top, **dict(how, bias=None if bias is None else torch.full((E,), 0.25, device="cuda")))
