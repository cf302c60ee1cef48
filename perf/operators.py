"""The operators around the packed linears, as cases with inputs, one pass, work and a definition in 64 bits.

Families ("kind"):
  norm     root-mean-square norm of a block's input with the residual's addition; the result in the activations' type, for a packed linear,
           or in e4m3 with a scale for each 128 columns, for an 8-bit one
  linear8  one linear whose weight is held in e4m3 with a scale for each 128x128 block: a module that a checkpoint leaves out of HTR-W1
  grouped  rows sorted by expert times their expert's matrix, 16-bit or in e4m3 with block scales, ragged
  experts  a routed-expert MLP on such stacked matrices, from the router's choice to the weighted sum

e4m3 values of a row are x / scale, rounded to nearest; the scale of each 128 columns is the least power of two that brings them to 448 or below,
so that the division is exact and what is rounded does not depend on how the scale was.
"""
import math
import random

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_F8 = torch.float8_e4m3fn
_BLOCK = 128
_LEAST = 2.0 ** -100      # amax of a block without values


def listed():
    return [
        # decode, one token: the norm in front of a packed linear
        dict(name="norm_1_row", kind="norm", rows=1, n=4096, dtype="bf16", residual=True, quantize=False),
        # a ragged prompt on a width that is no multiple of 128, float16
        dict(name="norm_333_rows_f16", kind="norm", rows=333, n=2824, dtype="f16", residual=True, quantize=False),
        # prefill: the norm whose result feeds an 8-bit linear
        dict(name="norm_8192_rows_e4m3", kind="norm", rows=8192, n=4096, dtype="bf16", residual=True, quantize=True),
        # decode, one token: the smallest linear of a layer, from 16-bit activations
        dict(name="k_proj8_1_row", kind="linear8", m=1024, n=4096, rows=1, dtype="bf16", pair=False, bias=False),
        # decode of 32 sequences: the largest linear of a layer, from the norm's 8-bit result
        dict(name="gate_up8_32_rows", kind="linear8", m=28672, n=4096, rows=32, dtype="bf16", pair=True, bias=False),
        # prefill of one ragged prompt, float16 with bias
        dict(name="qkv_proj8_333_rows", kind="linear8", m=6144, n=4096, rows=333, dtype="f16", pair=False, bias=True),
        # prefill of several prompts at once
        dict(name="gate_proj8_8192_rows", kind="linear8", m=14336, n=4096, rows=8192, dtype="bf16", pair=True, bias=False),
        # routed experts in decode: 16 tokens, top 6 of 64, gate and up in 8 bits
        dict(name="grouped8_96_rows", kind="grouped", experts=64, m=2816, n=2048, rows=96, dtype="bf16", bits=8),
        # routed experts in prefill: 500 tokens
        dict(name="grouped16_3000_rows", kind="grouped", experts=64, m=2816, n=2048, rows=3000, dtype="bf16", bits=16),
        # the down projection of 4096 tokens, float16, experts without rows among them
        dict(name="grouped16_24576_rows", kind="grouped", experts=64, m=2048, n=1408, rows=24576, dtype="f16", bits=16),
        # the whole layer in decode, 8 bits
        dict(name="experts8_16_tokens", kind="experts", tokens=16, experts=64, top=6, hidden=2048, inter=1408, dtype="bf16", bits=8),
        # the whole layer in prefill, 16 bits
        dict(name="experts16_4096_tokens", kind="experts", tokens=4096, experts=64, top=6, hidden=2048, inter=1408, dtype="bf16", bits=16),
    ]


def _log_uniform(rng, lo, hi):
    return math.exp(rng.uniform(math.log(lo), math.log(hi)))


def _size(rng, lo, hi, unit=1):
    """A log-uniform multiple of `unit` between lo and hi (both multiples of it)."""
    return min(hi, max(lo, unit * round(_log_uniform(rng, lo, hi) / unit)))


def draw(rng):
    most = [max(work(c)[k] for c in listed()) for k in ("bytes", "flops")]
    while True:
        kind = rng.choice(("norm", "linear8", "linear8", "grouped", "grouped", "experts"))
        dtype = rng.choice(("bf16", "bf16", "f16"))
        if kind == "norm":
            quantize = rng.random() < 0.5
            case = dict(kind=kind, rows=rng.choice((1, _size(rng, 1, 16384), _size(rng, 1, 16384))),
                        n=_size(rng, 128, 16384, 128) if quantize else _size(rng, 64, 16384, rng.choice((1, 8, 8, 128))),
                        dtype=rng.choice((dtype, dtype, "f32")), residual=rng.random() < 0.7, quantize=quantize)
        elif kind == "linear8":
            case = dict(kind=kind, m=_size(rng, 64, 28672, rng.choice((1, 32, 128))), n=_size(rng, 256, 14336, 128),
                        rows=rng.choice((1, _size(rng, 1, 64), _size(rng, 1, 8192), _size(rng, 65, 8192))), dtype=dtype,
                        pair=rng.random() < 0.5, bias=rng.random() < 0.3)
        elif kind == "grouped":
            bits = rng.choice((8, 16))
            case = dict(kind=kind, experts=rng.choice((1, 8, 16, 60, 64, 128)), m=_size(rng, 64, 8192, rng.choice((1, 32, 128))),
                        n=_size(rng, 256, 8192, 128) if bits == 8 else _size(rng, 256, 8192, 8), rows=_size(rng, 1, 32768), dtype=dtype, bits=bits)
        else:
            experts = rng.choice((8, 16, 32, 64, 128))
            case = dict(kind=kind, tokens=_size(rng, 1, 4096), experts=experts, top=rng.randint(1, min(8, experts // 2)),
                        hidden=_size(rng, 512, 4096, 128), inter=_size(rng, 256, 2048, 128), dtype=dtype, bits=rng.choice((8, 16)))
        w = work(case)
        if w["bytes"] <= most[0] and w["flops"] <= most[1]:
            return case


def _counts(case):
    """Rows of every expert, in descending order: popular and unpopular experts, the same for every seed."""
    rng = random.Random("%d %d" % (case["experts"], case["rows"]))
    share = sorted((math.exp(rng.gauss(0.0, 0.8)) for _ in range(case["experts"])), reverse=True)
    edges = [round(case["rows"] * sum(share[:i]) / sum(share)) for i in range(case["experts"] + 1)]
    return [b - a for a, b in zip(edges, edges[1:])]


def work(case):
    kind = case["kind"]
    size = 4 if case["dtype"] == "f32" else 2
    if kind == "norm":
        rows, n = case["rows"], case["n"]
        out = rows * n * (1 + 4 / _BLOCK) if case["quantize"] else rows * n * size
        return dict(bytes=rows * n * size * (3 if case["residual"] else 1) + n * size + out, flops=rows * n * 4)
    # bytes of an element of 8-bit rows or matrices, their scales among them
    row8, matrix8 = 1 + 4 / _BLOCK, 1 + 4 / _BLOCK ** 2
    if kind == "linear8":
        m, n, rows = case["m"], case["n"], case["rows"]
        return dict(bytes=rows * n * (row8 if case["pair"] else size) + m * n * matrix8 + rows * m * size + (m * size if case["bias"] else 0),
                    flops=2 * rows * m * n)
    if kind == "grouped":
        m, n, rows = case["m"], case["n"], case["rows"]
        active = sum(c > 0 for c in _counts(case))
        return dict(bytes=rows * n * (row8 if case["bits"] == 8 else size) + active * m * n * (matrix8 if case["bits"] == 8 else size)
                    + rows * m * size + 4 * case["experts"], flops=2 * rows * m * n)
    T, E, H, F, top = case["tokens"], case["experts"], case["hidden"], case["inter"], case["top"]
    active = E * (1 - (1 - top / E) ** T)      # expected; the choice is the seed's
    return dict(bytes=T * H * 2 * size + active * 3 * H * F * (matrix8 if case["bits"] == 8 else size) + T * top * 12, flops=6 * T * top * H * F)


# ---- inputs: everything is drawn on the GPU by one generator per state
def _block_scaled(w):
    """(e4m3 values, float32 scales) of matrices [..., m, n], one scale for each 128x128 block, the last rows' block may be shorter."""
    *lead, m, n = w.shape
    up = -(-m // _BLOCK)
    padded = torch.zeros(*lead, up * _BLOCK, n, device=w.device)
    padded[..., :m, :] = w
    blocks = padded.view(*lead, up, _BLOCK, n // _BLOCK, _BLOCK)
    scales = blocks.abs().amax(dim=(-3, -1)) / 448
    q = (blocks / scales[..., :, None, :, None]).to(_F8)
    return q.view(*lead, up * _BLOCK, n)[..., :m, :].contiguous(), scales.contiguous()


def _weight(gen, shape, dtype, bits):
    """Matrices whose rows and columns differ in size, as trained ones do."""
    m, n = shape[-2:]
    w = torch.randn(shape, device=gen.device, generator=gen)
    w *= torch.exp(0.3 * torch.randn(m, 1, device=gen.device, generator=gen)) * n ** -0.5
    return _block_scaled(w) if bits == 8 else w.to(_DTYPES[dtype])


def _activations(gen, rows, n, dtype):
    """Rows of unit size with a few columns that are much larger in all of them."""
    columns = torch.exp(0.5 * torch.randn(n, device=gen.device, generator=gen))
    return (torch.randn(rows, n, device=gen.device, generator=gen) * columns).to(_DTYPES[dtype])


def prepare(case, seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    gen = torch.Generator(device=dev).manual_seed(seed)
    kind, dtype = case["kind"], case["dtype"]
    if kind == "norm":
        x = _activations(gen, case["rows"], case["n"], dtype)
        residual = (3 * torch.randn(case["rows"], case["n"], device=dev, generator=gen)).to(x.dtype) if case["residual"] else None
        weight = (1 + 0.2 * torch.randn(case["n"], device=dev, generator=gen)).to(x.dtype)
        return dict(kind=kind, x=x, residual=residual, weight=weight, quantize=case["quantize"], eps=1e-6)
    if kind == "linear8":
        x = _activations(gen, case["rows"], case["n"], dtype)
        bias = torch.randn(case["m"], device=dev, generator=gen).to(x.dtype) if case["bias"] else None
        q, scales = _weight(gen, (case["m"], case["n"]), dtype, 8)
        return dict(kind=kind, x=_quantized(x.float()) if case["pair"] else x, q=q, scales=scales, bias=bias, dtype=x.dtype)
    if kind == "grouped":
        counts = torch.tensor(_counts(case))[torch.randperm(case["experts"], generator=torch.Generator().manual_seed(seed))]
        x = _activations(gen, case["rows"], case["n"], dtype)
        return dict(kind=kind, x=_quantized(x.float()) if case["bits"] == 8 else x, ends=counts.cumsum(0).to(torch.int32).to(dev),
                    weight=_weight(gen, (case["experts"], case["m"], case["n"]), dtype, case["bits"]), most=int(counts.max()), dtype=x.dtype)
    T, E, H, F = case["tokens"], case["experts"], case["hidden"], case["inter"]
    gate_up, down = _weight(gen, (E, 2 * F, H), dtype, case["bits"]), _weight(gen, (E, H, F), dtype, case["bits"])
    # a router with popular and unpopular experts; tokens prefer different ones
    logits = torch.randn(T, E, device=dev, generator=gen) + 0.5 * torch.randn(E, device=dev, generator=gen)
    probs, ids = torch.topk(torch.softmax(logits, dim=-1), case["top"], dim=-1)
    x = torch.randn(T, H, device=dev, generator=gen).to(_DTYPES[dtype])
    return dict(kind=kind, x=x, ids=ids, probs=probs / probs.sum(-1, keepdim=True), gate_up=gate_up, down=down,
                most=int(torch.bincount(ids.reshape(-1)).max()))


# ---- the plain forms
def _quantized(x):
    """(e4m3 values, float32 scales) of rows, one scale for each 128 columns: the least power of two from amax / 448 up."""
    blocks = x.unflatten(-1, (-1, _BLOCK))
    fraction, exponent = torch.frexp(blocks.abs().amax(-1).clamp(min=_LEAST))      # amax = fraction 2^exponent, 448 = 0.875 2^9
    scales = torch.ldexp(torch.ones_like(fraction), exponent - 9 + (fraction > 0.875))
    return (blocks / scales[..., None]).float().to(_F8).flatten(-2), scales.float()


def _rows(x):
    """Activations in float32, from either form."""
    return x[0].float() * x[1].repeat_interleave(_BLOCK, -1) if isinstance(x, tuple) else x.float()


def _matrix(w):
    """Matrices in float32, from either form."""
    if not isinstance(w, tuple):
        return w.float()
    q, scales = w
    return q.float() * scales.repeat_interleave(_BLOCK, -1).repeat_interleave(_BLOCK, -2)[..., :q.shape[-2], :]


def _by_expert(x, expert, place, w, most):
    """Row r of x times the matrix of expert[r], of which it is row number place[r]: one product of matrices padded to `most` rows."""
    padded = torch.zeros(w.shape[0], most, x.shape[1], device=x.device)
    padded[expert, place] = x
    return torch.bmm(padded, w.transpose(1, 2).contiguous())[expert, place]


def run(state):
    kind = state["kind"]
    if own:
        from htr_amd import ops
        if kind == "norm":
            return ops.rms_norm(state["x"], state["weight"], state["eps"], residual=state["residual"], quantize=state["quantize"])
        if kind == "linear8":
            return ops.linear_fp8(state["x"], state["q"], state["scales"], state["bias"], out_dtype=state["dtype"])
        if kind == "grouped":
            return ops.grouped_mm(state["x"], state["weight"], state["ends"], out_dtype=state["dtype"])
        return ops.moe_experts_stacked(state["x"], state["ids"], state["probs"], state["gate_up"], state["down"])
    x = state["x"]
    if kind == "norm":
        h = x.float()
        if state["residual"] is not None:
            total = (h + state["residual"].float()).to(x.dtype)
            h = total.float()
        if state["quantize"]:
            h = h.double()      # a scale next to a power of two
        y = h * torch.rsqrt((h * h).mean(-1, keepdim=True) + state["eps"]) * state["weight"].float()
        y = _quantized(y) if state["quantize"] else y.to(x.dtype)
        return y if state["residual"] is None else (y, total)
    if kind == "linear8":
        rows = x if isinstance(x, tuple) else _quantized(x.float())
        y = _rows(rows) @ _matrix((state["q"], state["scales"])).T
        return (y if state["bias"] is None else y + state["bias"].float()).to(state["dtype"])
    if kind == "grouped":
        rows = _rows(x)
        ends = state["ends"].long()
        row = torch.arange(rows.shape[0], device=rows.device)
        expert = torch.searchsorted(ends, row, right=True)
        start = torch.cat((ends.new_zeros(1), ends[:-1]))
        return _by_expert(rows, expert, row - start[expert], _matrix(state["weight"]), state["most"]).to(state["dtype"])
    T, top = state["ids"].shape
    eight = isinstance(state["gate_up"], tuple)
    expert, order = state["ids"].reshape(-1).sort(stable=True)
    place = torch.arange(T * top, device=x.device) - torch.searchsorted(expert, expert)
    rows = _rows(_quantized(x.float()) if eight else x)[order // top]
    gate, up = _by_expert(rows, expert, place, _matrix(state["gate_up"]), state["most"]).chunk(2, -1)
    hidden = gate / (1 + torch.exp(-gate)) * up
    out = _by_expert(_rows(_quantized(hidden)) if eight else hidden, expert, place, _matrix(state["down"]), state["most"])
    out = out * state["probs"].reshape(-1)[order][:, None]
    return out[order.argsort()].view(T, top, -1).sum(1).to(x.dtype)


# ---- the definitions in 64 bits
def _e4m3(v):
    """Float64 values to the nearest of e4m3, ties to even: three fraction bits, steps of 2^-9 below 2^-6."""
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6))) - 3)
    return (torch.round(v / step) * step).clamp(-448, 448)


def _quantized64(x):
    blocks = x.view(*x.shape[:-1], -1, _BLOCK)
    least = blocks.abs().amax(-1).clamp(min=_LEAST) / 448
    scales = torch.exp2(torch.floor(torch.log2(least)) - 1)
    for _ in range(3):
        scales = torch.where(scales < least, scales * 2, scales)
    return _e4m3(blocks / scales.unsqueeze(-1)).view(x.shape), scales


def _wide(q, scales, rows):
    """8-bit values of rows (rows = 1) or matrices (128) in 64 bits."""
    s = scales.double().repeat_interleave(_BLOCK, -1)
    return q.double() * (s if rows == 1 else s.repeat_interleave(rows, -2)[..., :q.shape[-2], :])


def exact(case, seed):
    s = prepare(case, seed)
    kind, x = case["kind"], s["x"]
    if kind == "norm":
        h = x.double()
        if case["residual"]:
            h = (x.double() + s["residual"].double()).to(x.dtype).double()      # one addition: what the stored sum is
        y = h / torch.sqrt((h * h).sum(-1, keepdim=True) / case["n"] + s["eps"]) * s["weight"].double()
        y = _quantized64(y) if case["quantize"] else y
        return (y, h) if case["residual"] else y
    if kind == "linear8":
        rows = _wide(*(x if case["pair"] else _quantized64(x.double())), 1)
        y = rows @ _wide(s["q"], s["scales"], _BLOCK).T
        return y + s["bias"].double() if case["bias"] else y

    def product(rows, w, e):
        return rows @ (_wide(w[0][e], w[1][e], _BLOCK) if case["bits"] == 8 else w[e].double()).T

    if kind == "grouped":
        y = torch.zeros(case["rows"], case["m"], dtype=torch.float64, device=s["ends"].device)
        first = 0
        for e, last in enumerate(s["ends"].tolist()):
            if last > first:
                rows = _wide(x[0][first:last], x[1][first:last], 1) if case["bits"] == 8 else x[first:last].double()
                y[first:last] = product(rows, s["weight"], e)
            first = last
        return y
    y = torch.zeros(case["tokens"], case["hidden"], dtype=torch.float64, device=x.device)
    rows = _wide(*_quantized64(x.double()), 1) if case["bits"] == 8 else x.double()
    for e in range(case["experts"]):
        token, slot = torch.nonzero(s["ids"] == e, as_tuple=True)
        if token.numel():
            g = product(rows[token], s["gate_up"], e)
            gate, up = g[:, :case["inter"]], g[:, case["inter"]:]
            hidden = gate * torch.sigmoid(gate) * up
            hidden = _wide(*_quantized64(hidden), 1) if case["bits"] == 8 else hidden
            y.index_add_(0, token, product(hidden, s["down"], e) * s["probs"][token, slot].double()[:, None])
    return y
