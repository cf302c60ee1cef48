"""Products in 8-bit integers and the router in front of routed experts, as cases with inputs, one pass, work and a definition in 64 bits.

Families ("kind"):
  route    a router's logits to each token's experts and their weights: softmax or sigmoid scores, a bias for balance, groups, renormalised weights
  norm     a block's norm with the residual's addition, rounded to int8 by row, and the int8 linear behind it
  linear   one linear whose weight is held in int8 with a scale for each channel, on rows in int8 with a scale for each token, or rounded to that
  grouped  rows in int8 sorted by expert times their expert's matrix in int8, ragged
  experts  a routed-expert MLP on such matrices, from the router's choice to the weighted sum

int8 values of a row are x / scale to the nearest integer, halves away from zero; the scale is the largest magnitude over 127, a float32.
"""
import math
import random

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_LEAST = 2.0 ** -100      # largest magnitude of a row without values


def listed():
    return [
        # decode, one token: the router of a layer with 64 experts, logits as a 16-bit linear leaves them
        dict(name="route_1_token", kind="route", tokens=1, experts=64, top=6, scores="softmax", bias=False, groups=1, top_groups=1, group_best=1, renormalize=True,
             dtype="bf16"),
        # a ragged prompt, 60 experts, scores that are not renormalised
        dict(name="route_500_tokens", kind="route", tokens=500, experts=60, top=4, scores="softmax", bias=False, groups=1, top_groups=1, group_best=1,
             renormalize=False, dtype="bf16"),
        # prefill: many experts in groups, sigmoid scores, a bias that balances the experts' load
        dict(name="route_16384_tokens", kind="route", tokens=16384, experts=256, top=8, scores="sigmoid", bias=True, groups=8, top_groups=4, group_best=2,
             renormalize=True, dtype="f32"),
        # decode, one token: norm and the queries', keys' and values' linear
        dict(name="norm_qkv_1_row", kind="norm", rows=1, m=6144, n=4096, dtype="bf16", residual=True, bias=False),
        # prefill of one ragged prompt, float16 with bias
        dict(name="norm_qkv_333_rows", kind="norm", rows=333, m=6144, n=4096, dtype="f16", residual=True, bias=True),
        # decode, one token: the smallest linear of a layer, from 16-bit activations
        dict(name="k_proj_1_row", kind="linear", m=1024, n=4096, rows=1, dtype="bf16", out="bf16", pair=False, bias=False),
        # decode of 8 sequences: the output head, float32 logits
        dict(name="lm_head_8_rows", kind="linear", m=152064, n=4096, rows=8, dtype="bf16", out="f32", pair=False, bias=False),
        # prefill of several prompts at once, from the norm's 8-bit result
        dict(name="gate_proj_8192_rows", kind="linear", m=14336, n=4096, rows=8192, dtype="bf16", out="bf16", pair=True, bias=False),
        # routed experts in decode: 16 tokens, top 6 of 64, gate and up
        dict(name="grouped_96_rows", kind="grouped", experts=64, m=2816, n=2048, rows=96, dtype="bf16"),
        # the down projection of 4096 tokens, float16, experts without rows among them
        dict(name="grouped_24576_rows", kind="grouped", experts=64, m=2048, n=1408, rows=24576, dtype="f16"),
        # the whole layer in decode
        dict(name="experts_16_tokens", kind="experts", tokens=16, experts=64, top=6, hidden=2048, inter=1408, dtype="bf16"),
        # the whole layer in prefill
        dict(name="experts_4096_tokens", kind="experts", tokens=4096, experts=64, top=6, hidden=2048, inter=1408, dtype="bf16"),
    ]


def _log_uniform(rng, lo, hi):
    return math.exp(rng.uniform(math.log(lo), math.log(hi)))


def _size(rng, lo, hi, unit=1):
    """A log-uniform multiple of `unit` between lo and hi (both multiples of it)."""
    return min(hi, max(lo, unit * round(_log_uniform(rng, lo, hi) / unit)))


def draw(rng):
    most = [max(work(c)[k] for c in listed()) for k in ("bytes", "flops")]
    while True:
        kind = rng.choice(("route", "route", "norm", "linear", "linear", "grouped", "grouped", "experts"))
        dtype = rng.choice(("bf16", "bf16", "f16"))
        if kind == "route":
            experts = rng.choice((8, 16, 60, 64, 72, 128, 160, 256, 384, 512))
            groups = rng.choice((1, 1, 4, 8)) if experts % 8 == 0 and experts >= 64 else 1
            top_groups = rng.randint(1, groups)
            case = dict(kind=kind, tokens=rng.choice((1, _size(rng, 1, 16384), _size(rng, 1, 16384))), experts=experts,
                        top=rng.randint(1, min(10, experts // 2, experts // groups * top_groups)), scores=rng.choice(("softmax", "sigmoid")), bias=rng.random() < 0.5,
                        groups=groups, top_groups=top_groups, group_best=rng.randint(1, 2), renormalize=rng.random() < 0.7, dtype=rng.choice((dtype, "f32")))
        elif kind in ("norm", "linear"):
            case = dict(kind=kind, m=_size(rng, 64, 28672, rng.choice((1, 32, 128))), n=_size(rng, 256, 14336, 16),
                        rows=rng.choice((1, _size(rng, 1, 64), _size(rng, 1, 8192), _size(rng, 65, 8192))), dtype=dtype, bias=rng.random() < 0.3)
            if kind == "norm":
                case.update(residual=rng.random() < 0.7)
            else:
                case.update(out=rng.choice((dtype, dtype, "f32")), pair=rng.random() < 0.5)
        elif kind == "grouped":
            case = dict(kind=kind, experts=rng.choice((1, 8, 16, 60, 64, 128)), m=_size(rng, 64, 8192, rng.choice((1, 32, 128))), n=_size(rng, 256, 8192, 16),
                        rows=_size(rng, 1, 32768), dtype=dtype)
        else:
            experts = rng.choice((8, 16, 32, 64, 128))
            case = dict(kind=kind, tokens=_size(rng, 1, 4096), experts=experts, top=rng.randint(1, min(8, experts // 2)), hidden=_size(rng, 512, 4096, 16),
                        inter=_size(rng, 256, 2048, 16), dtype=dtype)
        w = work(case)
        if w["bytes"] <= most[0] and w["flops"] <= most[1]:
            return case


def _counts(case):
    """Rows of every expert, in descending order: popular and unpopular experts, the same for every seed."""
    rng = random.Random("%d %d" % (case["experts"], case["rows"]))
    share = sorted((math.exp(rng.gauss(0.0, 0.8)) for _ in range(case["experts"])), reverse=True)
    edges = [round(case["rows"] * sum(share[:i]) / sum(share)) for i in range(case["experts"] + 1)]
    return [b - a for a, b in zip(edges, edges[1:])]


def _bytes_of(dtype):
    return 4 if dtype == "f32" else 2


def work(case):
    kind, size = case["kind"], _bytes_of(case["dtype"])
    if kind == "route":
        T, E, top = case["tokens"], case["experts"], case["top"]
        return dict(bytes=T * E * size + (4 * E if case["bias"] else 0) + T * top * 8, flops=T * E * 8)
    if kind in ("norm", "linear"):
        m, n, rows = case["m"], case["n"], case["rows"]
        matrix = m * n + 4 * m + (m * size if case["bias"] else 0)
        if kind == "norm":
            return dict(bytes=rows * n * size * (3 if case["residual"] else 1) + n * size + matrix + rows * m * size, flops=2 * rows * m * n + 4 * rows * n)
        return dict(bytes=(rows * (n + 4) if case["pair"] else rows * n * size) + matrix + rows * m * _bytes_of(case["out"]), flops=2 * rows * m * n)
    if kind == "grouped":
        m, n, rows = case["m"], case["n"], case["rows"]
        active = sum(c > 0 for c in _counts(case))
        return dict(bytes=rows * (n + 4) + active * m * (n + 4) + rows * m * size + 4 * case["experts"], flops=2 * rows * m * n)
    T, E, H, F, top = case["tokens"], case["experts"], case["hidden"], case["inter"], case["top"]
    active = E * (1 - (1 - top / E) ** T)      # expected; the choice is the seed's
    return dict(bytes=T * H * 2 * size + active * (3 * H * F + 8 * F + 4 * H) + T * top * 12, flops=6 * T * top * H * F)


# ---- inputs: everything is drawn on the GPU by one generator per state
def _weight(gen, *shape):
    """(int8 values, float32 scales) of matrices [..., m, n] whose rows and columns differ in size, as trained ones do."""
    m, n = shape[-2:]
    q = torch.empty(shape, dtype=torch.int8, device=gen.device)
    scales = torch.empty(shape[:-1], device=gen.device)
    columns = torch.exp(0.2 * torch.randn(n, device=gen.device, generator=gen))
    flat, s = q.view(-1, n), scales.view(-1)
    step = max(1, (1 << 28) // n)
    for i in range(0, flat.shape[0], step):      # in pieces, since float32 takes four times the matrix
        rows = torch.randn(min(step, flat.shape[0] - i), n, device=gen.device, generator=gen) * columns
        rows *= torch.exp(0.3 * torch.randn(rows.shape[0], 1, device=gen.device, generator=gen)) * n ** -0.5
        s[i:i + step] = rows.abs().amax(-1) / 127
        flat[i:i + step] = (rows / s[i:i + step, None]).round().to(torch.int8)
    return q, scales


def _activations(gen, rows, n, dtype):
    """Rows of unit size with a few columns that are much larger in all of them."""
    columns = torch.exp(0.5 * torch.randn(n, device=gen.device, generator=gen))
    return (torch.randn(rows, n, device=gen.device, generator=gen) * columns).to(_DTYPES[dtype])


def prepare(case, seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    gen = torch.Generator(device=dev).manual_seed(seed)
    kind, dtype = case["kind"], case["dtype"]
    if kind == "route":
        # popular and unpopular experts; the bias works against what makes them so
        popular = 0.5 * torch.randn(case["experts"], device=dev, generator=gen)
        logits = (1.5 * torch.randn(case["tokens"], case["experts"], device=dev, generator=gen) + popular).to(_DTYPES[dtype])
        bias = -0.1 * popular + 0.01 * torch.randn(case["experts"], device=dev, generator=gen) if case["bias"] else None
        return dict(kind=kind, logits=logits, bias=bias, top=case["top"], scores=case["scores"], groups=case["groups"], top_groups=case["top_groups"],
                    group_best=case["group_best"], renormalize=case["renormalize"], scale=2.5 if case["scores"] == "sigmoid" else 1.0)
    if kind in ("norm", "linear"):
        x = _activations(gen, case["rows"], case["n"], dtype)
        q, scales = _weight(gen, case["m"], case["n"])
        bias = torch.randn(case["m"], device=dev, generator=gen).to(_DTYPES[case.get("out", dtype)]) if case["bias"] else None
        if kind == "linear":
            return dict(kind=kind, x=_quantized(x) if case["pair"] else x, q=q, scales=scales, bias=bias, dtype=_DTYPES[case["out"]])
        residual = (3 * torch.randn(case["rows"], case["n"], device=dev, generator=gen)).to(x.dtype) if case["residual"] else None
        weight = (1 + 0.2 * torch.randn(case["n"], device=dev, generator=gen)).to(x.dtype)
        return dict(kind=kind, x=x, residual=residual, weight=weight, eps=1e-6, q=q, scales=scales, bias=bias, dtype=x.dtype)
    if kind == "grouped":
        counts = torch.tensor(_counts(case))[torch.randperm(case["experts"], generator=torch.Generator().manual_seed(seed))]
        return dict(kind=kind, x=_quantized(_activations(gen, case["rows"], case["n"], dtype)), ends=counts.cumsum(0).to(torch.int32).to(dev),
                    weight=_weight(gen, case["experts"], case["m"], case["n"]), most=int(counts.max()), dtype=_DTYPES[dtype])
    T, E, H, F = case["tokens"], case["experts"], case["hidden"], case["inter"]
    gate_up, down = _weight(gen, E, 2 * F, H), _weight(gen, E, H, F)
    # a router with popular and unpopular experts; tokens prefer different ones
    logits = torch.randn(T, E, device=dev, generator=gen) + 0.5 * torch.randn(E, device=dev, generator=gen)
    probs, ids = torch.topk(torch.softmax(logits, dim=-1), case["top"], dim=-1)
    x = torch.randn(T, H, device=dev, generator=gen).to(_DTYPES[dtype])
    return dict(kind=kind, x=x, ids=ids, probs=probs / probs.sum(-1, keepdim=True), gate_up=gate_up, down=down, most=int(torch.bincount(ids.reshape(-1)).max()))


# ---- the plain forms
def _quantized(x):
    """(int8 values, float32 scales) of rows: quotients in 64 bits, since a half decides between two integers."""
    scales = (x.abs().amax(-1).double().clamp(min=_LEAST) / 127).float()
    z = x.double() / scales.double()[..., None]
    return (torch.sign(z) * torch.floor(z.abs() + 0.5)).to(torch.int8), scales


def _product(rows, q, scales):
    """Rows (values, scales) times one matrix, in float32."""
    return (rows[0].float() @ q.float().T) * rows[1][:, None] * scales


def _by_expert(rows, expert, place, w, most):
    """Row r times the matrix of expert[r], of which it is row number place[r]: one product of matrices padded to `most` rows."""
    padded = torch.zeros(w[0].shape[0], most, rows[0].shape[1], device=rows[0].device)
    padded[expert, place] = rows[0].float()
    return torch.bmm(padded, w[0].float().transpose(1, 2).contiguous())[expert, place] * rows[1][:, None] * w[1][expert]


def _route(s):
    logits = s["logits"].double()      # 64 bits: scores next to each other
    if s["scores"] == "softmax":
        e = torch.exp(logits - logits.amax(-1, keepdim=True))
        scores = e / e.sum(-1, keepdim=True)
    else:
        scores = 1 / (1 + torch.exp(-logits))
    # without a bias the scores' order is the logits'
    rank = logits if s["bias"] is None else scores + s["bias"].double()
    if s["groups"] > 1:
        by_group = (scores if s["bias"] is None and s["group_best"] > 1 else rank).unflatten(-1, (s["groups"], -1))
        best = by_group.sort(dim=-1, descending=True).values[..., :s["group_best"]].sum(-1)
        chosen = best.sort(dim=-1, descending=True, stable=True).indices[..., :s["top_groups"]]
        out = torch.ones_like(best, dtype=torch.bool).scatter(-1, chosen, False)
        rank = rank.masked_fill(out.repeat_interleave(by_group.shape[-1], -1), -torch.inf)
    ids = rank.sort(dim=-1, descending=True, stable=True).indices[..., :s["top"]]
    weights = scores.gather(-1, ids)
    if s["renormalize"]:
        weights = weights / weights.sum(-1, keepdim=True)
    return ids.to(torch.int32), (weights * s["scale"]).float()


def run(state):
    kind = state["kind"]
    if own:
        from htr_amd import ops
        if kind == "route":
            return ops.route_experts(state["logits"], state["top"], scores=state["scores"], bias=state["bias"], groups=state["groups"],
                                     top_groups=state["top_groups"], group_best=state["group_best"], renormalize=state["renormalize"], scale=state["scale"])
        if kind == "norm":
            out = ops.rms_norm(state["x"], state["weight"], state["eps"], residual=state["residual"], quantize=torch.int8)
            rows, total = out if state["residual"] is not None else (out, None)
            y = ops.linear_int8(rows, state["q"], state["scales"], state["bias"], out_dtype=state["dtype"])
            return y if total is None else (y, total)
        if kind == "linear":
            return ops.linear_int8(state["x"], state["q"], state["scales"], state["bias"], out_dtype=state["dtype"])
        if kind == "grouped":
            return ops.grouped_mm(state["x"], state["weight"], state["ends"], out_dtype=state["dtype"])
        return ops.moe_experts_stacked(state["x"], state["ids"], state["probs"], state["gate_up"], state["down"])
    if kind == "route":
        return _route(state)
    x = state["x"]
    if kind in ("norm", "linear"):
        total = None
        if kind == "linear":
            rows = x if isinstance(x, tuple) else _quantized(x)
        else:
            t = x
            if state["residual"] is not None:
                t = total = (x.float() + state["residual"].float()).to(x.dtype)
            h = t.double()      # 64 bits: halves again
            rows = _quantized(h / torch.sqrt((h * h).mean(-1, keepdim=True) + state["eps"]) * state["weight"].double())
        y = _product(rows, state["q"], state["scales"])
        y = (y if state["bias"] is None else y + state["bias"].float()).to(state["dtype"])
        return y if total is None else (y, total)
    if kind == "grouped":
        ends = state["ends"].long()
        row = torch.arange(x[0].shape[0], device=ends.device)
        expert = torch.searchsorted(ends, row, right=True)
        start = torch.cat((ends.new_zeros(1), ends[:-1]))
        return _by_expert(x, expert, row - start[expert], state["weight"], state["most"]).to(state["dtype"])
    T, top = state["ids"].shape
    expert, order = state["ids"].reshape(-1).sort(stable=True)
    place = torch.arange(T * top, device=x.device) - torch.searchsorted(expert, expert)
    q, scales = _quantized(x)
    gate, up = _by_expert((q[order // top], scales[order // top]), expert, place, state["gate_up"], state["most"]).chunk(2, -1)
    out = _by_expert(_quantized(gate / (1 + torch.exp(-gate)) * up), expert, place, state["down"], state["most"])
    out = out * state["probs"].reshape(-1)[order][:, None]
    return out[order.argsort()].view(T, top, -1).sum(1).to(x.dtype)


# ---- the definitions in 64 bits
def _rows64(x):
    """(integers, scales) of rows, both float64."""
    scales = (x.abs().max(-1, keepdim=True).values.clamp(min=_LEAST) / 127).float().double()
    return torch.trunc(x / scales + torch.copysign(torch.full_like(x, 0.5), x)), scales


def _wide(pair):
    return pair[0].double() * pair[1].double().unsqueeze(-1)


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "route":
        l = s["logits"].double()
        scores = torch.softmax(l, -1) if case["scores"] == "softmax" else torch.sigmoid(l)
        rank = scores + s["bias"].double() if case["bias"] else l
        if case["groups"] > 1:
            by = (rank if case["bias"] or case["group_best"] == 1 else scores).view(case["tokens"], case["groups"], -1)
            best = torch.topk(by, case["group_best"], dim=-1).values.sum(-1)
            # a group is in where fewer than top_groups others are better, or as good and before it
            before = torch.arange(case["groups"], device=l.device)
            better = (best[:, None, :] > best[:, :, None]) | ((best[:, None, :] == best[:, :, None]) & (before[None, None, :] < before[None, :, None]))
            rank = torch.where((better.sum(-1) < case["top_groups"]).unsqueeze(-1).expand_as(by).reshape(rank.shape), rank, -torch.inf)
        ids = torch.sort(-rank, dim=-1, stable=True).indices[:, :case["top"]]
        weights = torch.take_along_dim(scores, ids, -1)
        return ids, weights / (weights.sum(-1, keepdim=True) if case["renormalize"] else 1) * s["scale"]
    if kind in ("norm", "linear"):
        total = None
        if kind == "linear" and case["pair"]:
            rows = _wide(s["x"])
        elif kind == "linear":
            rows = torch.mul(*_rows64(s["x"].double()))
        else:
            total = s["x"].double()
            if case["residual"]:
                total = (total + s["residual"].double()).to(s["x"].dtype).double()      # one addition: what the stored sum is
            norm = torch.sqrt(total.square().sum(-1, keepdim=True) / case["n"] + s["eps"])
            rows = torch.mul(*_rows64(total / norm * s["weight"].double()))
        y = rows @ _wide((s["q"], s["scales"])).T
        y = y + s["bias"].double() if case["bias"] else y
        return (y, total) if kind == "norm" and case["residual"] else y
    if kind == "grouped":
        y = torch.zeros(case["rows"], case["m"], dtype=torch.float64, device=s["ends"].device)
        first = 0
        for e, last in enumerate(s["ends"].tolist()):
            if last > first:
                y[first:last] = _wide((s["x"][0][first:last], s["x"][1][first:last])) @ _wide((s["weight"][0][e], s["weight"][1][e])).T
            first = last
        return y
    y = torch.zeros(case["tokens"], case["hidden"], dtype=torch.float64, device=s["x"].device)
    rows = torch.mul(*_rows64(s["x"].double()))
    for e in range(case["experts"]):
        token, slot = torch.nonzero(s["ids"] == e, as_tuple=True)
        if token.numel():
            g = rows[token] @ _wide((s["gate_up"][0][e], s["gate_up"][1][e])).T
            gate, up = g[:, :case["inter"]], g[:, case["inter"]:]
            hidden = torch.mul(*_rows64(gate * torch.sigmoid(gate) * up))
            y.index_add_(0, token, hidden @ _wide((s["down"][0][e], s["down"][1][e])).T * s["probs"][token, slot].double()[:, None])
    return y
