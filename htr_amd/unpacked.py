"""The operators around the packed linears: the norm in front of them, linears and routed experts that a checkpoint leaves out of HTR-W1, and the experts' router.

    y, h = ops.rms_norm(x, weight, residual=h)                           # 16-bit result, for ops.linear
    xq, h = ops.rms_norm(x, weight, residual=h, quantize=True)           # (e4m3 values, scales), for the two below
    y = ops.linear_fp8(xq, qweight, scales)                              # weight in e4m3 with a scale for each 128x128 block
    xq, h = ops.rms_norm(x, weight, residual=h, quantize=torch.int8)     # (int8 values, scales)
    y = ops.linear_int8(xq, qweight, scales)                             # weight in int8 with a scale for each channel
    y = ops.grouped_mm(xs, weights, ends)                                # rows sorted by expert, stacked matrices in 16 or 8 bits
    ids, weights = ops.route_experts(logits, 6)                          # a router's logits, for ops.moe_experts and
    y = ops.moe_experts_stacked(x, ids, weights, gate_up, down)          # ops.moe_experts on such matrices

The reference leaves these modules to its caller (its plugin returns UnquantizedLinearMethod, htr/vllm_plugin.py:49-69).

8-bit rows are a pair (values float8_e4m3fn [..., n], scales float32 [..., n / 128]), 8-bit matrices a pair (values [.., m, n], scales
[.., ceil(m / 128), n / 128]); a value stands for itself times its block's scale.  The scales made here are powers of two, the least that brings
the block to 448 or below; scales from elsewhere need not be.  Infinities and NaN become NaN.

In int8 a row has one scale: rows are (values int8 [..., n], scales float32 [...]), matrices (values [.., m, n], scales [.., m]), n a multiple of 16.  The
scales made here are the row's largest magnitude over 127, the values the nearest integers, halves away from zero; a row with an infinity or NaN has the scale NaN.

Norms sum in 64 bits, products of 16-bit values in float32.  Products of e4m3 values are first added eight consecutive
columns at a time, as the matrix instructions do: each eight is off by at most 2^-10 of the largest magnitude in x times that in the matrix (one below 2^-6 of its
scale counts as that).  Sums of int8 products are exact; one is multiplied with its row's scale, then with its channel's.
Everything beyond is float32, the product of a row's scale and a block's as well (below 2^-126 it has fewer bits, beyond float32 it is
infinite).  Results are rounded once.  Nothing here has a derivative, as no packed linear has one in its
activations: a call that torch would differentiate is refused.  Calls only queue kernels on the current stream of x's device, allocate with torch and
may be captured into a graph.
"""
import torch

from . import _native

E4M3, I8 = torch.float8_e4m3fn, torch.int8
_CODE = {torch.bfloat16: _native.BF16, torch.float16: _native.F16, torch.float32: _native.F32, E4M3: _native.E4M3, I8: _native.I8}
_UNIT = {E4M3: 128, I8: 16}      # columns of 8-bit rows come in
_HALVES = (torch.bfloat16, torch.float16)
_FLOATS = (torch.bfloat16, torch.float16, torch.float32)

_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda index: torch.cuda.current_stream(index).cuda_stream)


def _refuse_derivatives(what, *tensors):
    for t in tensors:
        if t is not None and ((t.requires_grad and torch.is_grad_enabled()) or torch._C._functorch.is_functorch_wrapped_tensor(t)
                              or torch.autograd.forward_ad._current_level >= 0):
            raise RuntimeError(f"{what} has no derivative: call it under torch.no_grad(), or on detached tensors")


def _fast(x):
    """(the C++ host path, the current stream of x's device), or None where there is none for it: tracers' tensors, the CPU."""
    if type(x) is not torch.Tensor or torch.compiler.is_compiling():
        return None
    index = x.get_device()
    if index < 0:
        return None
    fast = _native.fast()
    return None if fast is None else (fast, _raw_stream(index))


def _on_one_gpu(what, first, *others):
    if not first.is_cuda:
        raise RuntimeError(f"{what} runs on a ROCm device only; move the tensors to the GPU")
    for t in others:
        if t is not None and t.device != first.device:
            raise RuntimeError(f"{what}: every tensor must be on the device of x")


def _rows(x):
    """(x as rows [M, n] with consecutive columns, elements from row to row)."""
    n = x.shape[-1]
    if x.dim() != 2:
        x = x.reshape(-1, n)
    if x.shape[1] != 1 and x.stride(1) != 1:
        x = x.contiguous()
    return x, x.stride(0) if x.shape[0] > 1 else n


def _packed(t):
    """t in consecutive memory from a 16-byte boundary on."""
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _queue(device, name, *args):
    with torch.cuda.device(device):
        _native.check(getattr(_native.lib(), name)(*args, _raw_stream(device.index)))


def rms_norm(x, weight, eps=1e-6, residual=None, quantize=False):
    """t = x + residual (rounded to x's type), y = t / sqrt(mean(t^2) + eps) * weight over the last dimension.

    x [..., n] and residual bfloat16, float16 or float32, weight [n] of the same type.  Returns y in x's type, or with quantize=True the pair
    (values, scales) of y in e4m3 (n a multiple of 128), with quantize=torch.int8 in int8 (n a multiple of 16); with a residual, (that, t): t is the next
    block's residual."""
    if isinstance(quantize, torch.dtype) and quantize not in _UNIT:
        raise RuntimeError("rms_norm: the result is rounded to torch.float8_e4m3fn (or True) or to torch.int8")
    kind = I8 if quantize is I8 else E4M3 if quantize else None
    path = _fast(x)
    if path is not None:
        y = path[0].rms_norm(x, weight, eps, residual, 2 if kind is I8 else int(kind is E4M3), path[1])
        if y is not None:
            return y
    if x.dim() < 1 or x.dtype not in _FLOATS or weight.dtype != x.dtype or weight.shape != x.shape[-1:]:
        raise RuntimeError("rms_norm wants x [..., n] in bfloat16, float16 or float32 and a weight [n] of that type")
    if residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype):
        raise RuntimeError("rms_norm: the residual must have x's shape and type")
    n = x.shape[-1]
    if n < 1 or (kind and n % _UNIT[kind]):
        raise RuntimeError("rms_norm: at least one column, and a multiple of 128 for an 8-bit result (16 in int8)")
    _on_one_gpu("rms_norm", x, weight, residual)
    _refuse_derivatives("rms_norm", x, weight, residual)
    x2, xs = _rows(x)
    r2, rs = (None, 0) if residual is None else _rows(residual)
    w = weight.contiguous()
    y = torch.empty(x.shape, dtype=kind or x.dtype, device=x.device)
    scales = torch.empty(_scales_shape(x.shape, kind), dtype=torch.float32, device=x.device) if kind else None
    total = None if residual is None else torch.empty(x.shape, dtype=x.dtype, device=x.device)
    if x.numel():
        _queue(x.device, "htr_rms_norm_int8" if kind is I8 else "htr_rms_norm", x2.data_ptr(), xs, _ptr(r2), rs, w.data_ptr(), x2.shape[0], n, eps, _CODE[x.dtype], y.data_ptr(),
               _ptr(scales), _ptr(total))
    out = (y, scales) if kind else y
    return out if residual is None else (out, total)


def _ptr(t):
    return None if t is None else t.data_ptr()


def _scales_shape(shape, kind):
    """Of 8-bit rows."""
    return shape[:-1] if kind is I8 else shape[:-1] + (shape[-1] // 128,)


def quantize_fp8(x):
    """(values, scales) of rows x [..., n] in e4m3, n a multiple of 128: what linear_fp8 and grouped_mm make of 16-bit rows by themselves."""
    if x.dim() < 1 or x.dtype not in _FLOATS or x.shape[-1] < 1 or x.shape[-1] % 128:
        raise RuntimeError("quantize_fp8 wants x [..., n] in bfloat16, float16 or float32, n a multiple of 128")
    _on_one_gpu("quantize_fp8", x)
    _refuse_derivatives("quantize_fp8", x)
    n = x.shape[-1]
    x2, stride = _rows(x)
    if x2.data_ptr() % 16 or stride % 8:
        x2, stride = x2.clone(memory_format=torch.contiguous_format), n
    q = torch.empty(x.shape, dtype=E4M3, device=x.device)
    scales = torch.empty(x.shape[:-1] + (n // 128,), dtype=torch.float32, device=x.device)
    if x.numel():
        _queue(x.device, "htr_quantize_e4m3", x2.data_ptr(), stride, x2.shape[0], n, _CODE[x.dtype], q.data_ptr(), scales.data_ptr())
    return q, scales


def quantize_int8(x):
    """(values, scales) of rows x [..., n] in int8, n a multiple of 16: what linear_int8 and grouped_mm make of floating rows by themselves."""
    if x.dim() < 1 or x.dtype not in _FLOATS or x.shape[-1] < 1 or x.shape[-1] % 16:
        raise RuntimeError("quantize_int8 wants x [..., n] in bfloat16, float16 or float32, n a multiple of 16")
    _on_one_gpu("quantize_int8", x)
    _refuse_derivatives("quantize_int8", x)
    x2, stride = _rows(x)
    q = torch.empty(x.shape, dtype=I8, device=x.device)
    scales = torch.empty(x.shape[:-1], dtype=torch.float32, device=x.device)
    if x.numel():
        _queue(x.device, "htr_quantize_int8", x2.data_ptr(), stride, x2.shape[0], x.shape[-1], _CODE[x.dtype], q.data_ptr(), scales.data_ptr())
    return q, scales


def quantize_weight_int8(w):
    """(values, scales) of matrices [.., m, n] in int8 with a scale for each of their rows (channels), n a multiple of 16, as quantize_int8 rounds.  Torch
    operations, on the CPU as well: for laying out a weight once."""
    if w.dim() < 2 or w.shape[-2] < 1 or w.shape[-1] < 1 or w.shape[-1] % 16:
        raise RuntimeError("quantize_weight_int8 wants matrices [.., m, n], n a multiple of 16")
    w = w.detach()
    amax = w.abs().amax(-1).double()
    scales = (amax.clamp(min=2.0 ** -100) / 127).float()
    ok = scales.isfinite()
    z = torch.where(ok[..., None], w.double() / scales.double()[..., None], 0.0)
    return (torch.sign(z) * torch.floor(z.abs() + 0.5)).to(I8), torch.where(ok, scales, torch.nan)


def dequantize_int8(q, scales):
    """float32 values of int8 rows or matrices."""
    return q.float() * scales[..., None]


def quantize_weight_fp8(w):
    """(values, scales) of matrices [.., m, n] in e4m3 with a scale for each 128x128 block (the last rows' blocks may be shorter), n a multiple
    of 128.  Torch operations, on the CPU as well: for laying out a weight once."""
    if w.dim() < 2 or w.shape[-2] < 1 or w.shape[-1] < 1 or w.shape[-1] % 128:
        raise RuntimeError("quantize_weight_fp8 wants matrices [.., m, n], n a multiple of 128")
    m, n = w.shape[-2:]
    up = -(-m // 128)
    padded = torch.zeros(w.shape[:-2] + (up * 128, n), dtype=torch.float32, device=w.device)
    padded[..., :m, :] = w.detach()
    padded = torch.where(padded.isfinite(), padded, torch.nan).unflatten(-2, (up, 128)).unflatten(-1, (n // 128, 128))
    fraction, exponent = torch.frexp(padded.abs().nan_to_num(0.0).amax(dim=(-3, -1)).clamp(min=2.0 ** -100))
    scales = torch.ldexp(torch.ones_like(fraction), exponent - 9 + (fraction > 0.875))
    q = (padded / scales[..., :, None, :, None]).to(E4M3)
    return q.flatten(-2).flatten(-3, -2)[..., :m, :].contiguous(), scales.contiguous()


def dequantize_fp8(q, scales):
    """float32 values of 8-bit rows or matrices, as linear_fp8 takes them (which of the two, the scales' shape says)."""
    s = scales.repeat_interleave(128, -1)
    if scales.shape[:-1] != q.shape[:-1] or q.dim() != scales.dim():
        s = s.repeat_interleave(128, -2)[..., :q.shape[-2], :]
    return q.float() * s


def _pair(x):
    """Whether x is a pair (values, scales); half a pair is refused."""
    if not isinstance(x, (tuple, list)):
        return False
    if len(x) != 2 or not isinstance(x[0], torch.Tensor) or not isinstance(x[1], torch.Tensor):
        raise RuntimeError("8-bit rows and matrices are pairs (values, scales) of tensors")
    return True


def _check_rows(what, x, experts, grouped, kind=E4M3):
    """x as htr_product takes it with an 8-bit weight: contiguous 8-bit rows (values, scales), to which a tensor is rounded, or few floating rows (x, None)."""
    if kind is I8:
        n = x.shape[-1] if isinstance(x, torch.Tensor) else 0
        if n and not grouped and x.dtype in _FLOATS and n % 16 == 0 and _native.lib().htr_product_rounds_int8(x.numel() // n, n):
            return _packed(x), None
        q, s = x if _pair(x) else quantize_int8(x)
        if q.dtype != I8 or s.dtype != torch.float32 or q.dim() < 1 or s.shape != q.shape[:-1] or q.shape[-1] % 16:
            raise RuntimeError(f"{what}: 8-bit rows for an int8 weight are (int8 [..., n], float32 [...]), n a multiple of 16")
        return _packed(q), s.contiguous()
    if not _pair(x):
        n = x.shape[-1]
        if x.dtype in _HALVES and n % 128 == 0 and n and _native.lib().htr_product_rounds(x.numel() // n, experts, int(grouped)):
            return _packed(x), None
        return quantize_fp8(x)
    q, s = x
    if q.dtype != E4M3 or s.dtype != torch.float32 or q.dim() < 1 or s.shape != q.shape[:-1] + (q.shape[-1] // 128,) or q.shape[-1] % 128:
        raise RuntimeError(f"{what}: 8-bit rows are (float8_e4m3fn [..., n], float32 [..., n / 128]), n a multiple of 128")
    return _packed(q), s.contiguous()


def _check_matrix(what, q, s, dims, kind=E4M3):
    if kind is I8:
        if not isinstance(q, torch.Tensor) or not isinstance(s, torch.Tensor) or q.dtype != I8 or s.dtype != torch.float32 or q.dim() != dims or q.shape[-1] % 16 or 0 in q.shape \
                or s.shape != q.shape[:-1] or q.shape[-1] >= 1 << 17:
            raise RuntimeError(f"{what}: an 8-bit weight in int8 is (int8 [.., m, n], float32 [.., m]), n a multiple of 16 below 131072")
    elif not isinstance(q, torch.Tensor) or not isinstance(s, torch.Tensor) or q.dtype != E4M3 or s.dtype != torch.float32 or q.dim() != dims or q.shape[-1] % 128 or 0 in q.shape \
            or s.shape != q.shape[:-2] + (-(-q.shape[-2] // 128), q.shape[-1] // 128):
        raise RuntimeError(f"{what}: an 8-bit weight is (float8_e4m3fn [.., m, n], float32 [.., ceil(m / 128), n / 128]), n a multiple of 128")
    if not q.is_contiguous() or not s.is_contiguous() or q.data_ptr() % 16:
        raise RuntimeError(f"{what}: weights must be contiguous, on a 16-byte boundary")


def _out_dtype(what, out_dtype, x, bias=None):
    if out_dtype is None:
        out_dtype = x.dtype if not _pair(x) else torch.bfloat16 if bias is None else bias.dtype
    if out_dtype not in _FLOATS:
        raise RuntimeError(f"{what}: the result is bfloat16, float16 or float32")
    return out_dtype


def _product(x, w, ws, bias, ends, out_dtype):
    """The common case of the products in C++; None where something else is asked for, or is wrong."""
    q, s = x if type(x) is tuple and len(x) == 2 and x[1] is not None else (x, None)
    path = _fast(q)
    if path is None:
        return None
    if out_dtype is None:
        out_dtype = q.dtype if s is None else torch.bfloat16 if bias is None else bias.dtype
    return path[0].product(q, s, w, ws, bias, ends, _CODE.get(out_dtype, -1), path[1])


def linear_fp8(x, qweight, scales, bias=None, out_dtype=None):
    """y = x @ W^T (+ bias), W [m, n] in e4m3 with a float32 scale for each 128x128 block, any m.

    x: [..., n] in bfloat16, float16 or float32, which is rounded to e4m3 for each 128 columns, or 8-bit rows (values, scales) as rms_norm and quantize_fp8
    give them.  y is of x's type; for 8-bit rows of the bias's, or bfloat16, unless out_dtype says."""
    if isinstance(qweight, torch.Tensor) and qweight.dtype is E4M3:
        y = _product(x, qweight, scales, bias, None, out_dtype)
        if y is not None:
            return y
    return _linear_8bit("linear_fp8", E4M3, x, qweight, scales, bias, out_dtype)


def _linear_8bit(what, kind, x, qweight, scales, bias, out_dtype):
    _check_matrix(what, qweight, scales, 2, kind)
    m, n = qweight.shape
    dtype = _out_dtype(what, out_dtype, x, bias)
    first = x[0] if _pair(x) else x
    if first.dim() < 1 or first.shape[-1] != n:
        raise RuntimeError(f"{what}: x has {first.shape[-1] if first.dim() else 0} columns, the weight {n}")
    if bias is not None and (bias.dtype != dtype or bias.shape != (m,)):
        raise RuntimeError(f"{what}: the bias must be [m] in the result's type")
    _on_one_gpu(what, first, qweight, scales, bias, x[1] if _pair(x) else None)
    _refuse_derivatives(what, *(x if _pair(x) else (x,)), qweight, scales, bias)
    q, s = _check_rows(what, x, 1, False, kind)
    bias = None if bias is None else bias.contiguous()
    y = torch.empty(first.shape[:-1] + (m,), dtype=dtype, device=q.device)
    if y.numel():
        _queue(q.device, "htr_product", q.data_ptr(), _CODE[q.dtype], _ptr(s), qweight.data_ptr(), scales.data_ptr(), _ptr(bias), None, y.data_ptr(), y.numel() // m,
               m, n, 1, _CODE[kind], _CODE[dtype])
    return y


def linear_int8(x, qweight, scales, bias=None, out_dtype=None):
    """y = x @ W^T (+ bias), W [m, n] in int8 with a float32 scale for each of its rows [m], any m, n a multiple of 16.

    x: [..., n] in bfloat16, float16 or float32, which is rounded to int8 row by row, or int8 rows (values, scales) as rms_norm and quantize_int8
    give them.  y is of x's type; for int8 rows of the bias's, or bfloat16, unless out_dtype says."""
    if isinstance(qweight, torch.Tensor) and qweight.dtype is I8:
        y = _product(x, qweight, scales, bias, None, out_dtype)
        if y is not None:
            return y
    return _linear_8bit("linear_int8", I8, x, qweight, scales, bias, out_dtype)


def grouped_mm(x, weight, ends, out_dtype=None):
    """Rows sorted by expert times their expert's matrix: y[r] = W_e x[r] for ends[e - 1] <= r < ends[e] (from 0).

    weight: [E, m, n] in bfloat16 or float16, x [R, n] of the same type, n a multiple of 8; or an 8-bit pair (values [E, m, n], scales), with x in
    8-bit rows of that kind (e4m3 or int8) or rounded to them.  ends: int32 [E] on the device (the running sum of the experts' row counts); an end below an earlier one counts as
    that one, one beyond R as R; rows from the last end on become zeros.  y [R, m] in x's type (8-bit rows: bfloat16) unless out_dtype says."""
    eight = _pair(weight)
    if ends is not None:
        y = _product(x, weight[0], weight[1], None, ends, out_dtype) if eight else _product(x, weight, None, None, ends, out_dtype)
        if y is not None:
            return y
    first = x[0] if _pair(x) else x
    if eight:
        w, ws = weight
        kind = I8 if w.dtype is I8 else E4M3
        _check_matrix("grouped_mm", w, ws, 3, kind)
    else:
        w, ws = weight, None
        if w.dtype not in _HALVES or w.dim() != 3 or w.shape[2] % 8 or 0 in w.shape:
            raise RuntimeError("grouped_mm: a 16-bit weight is bfloat16 or float16 [E, m, n], n a multiple of 8")
        if not w.is_contiguous() or w.data_ptr() % 16:
            raise RuntimeError("grouped_mm: weights must be contiguous, on a 16-byte boundary")
        if _pair(x) or x.dtype != w.dtype:
            raise RuntimeError("grouped_mm: x must be of the weight's type")
    E, m, n = w.shape
    dtype = _out_dtype("grouped_mm", out_dtype, x)
    if first.dim() != 2 or first.shape[1] != n:
        raise RuntimeError(f"grouped_mm wants rows [R, {n}]")
    if ends is None or ends.dtype != torch.int32 or ends.shape != (E,):
        raise RuntimeError("grouped_mm: ends must be int32, one for each expert")
    _on_one_gpu("grouped_mm", first, w, ws, ends, x[1] if _pair(x) else None)
    _refuse_derivatives("grouped_mm", *(x if _pair(x) else (x,)), w, ws)
    q, s = _check_rows("grouped_mm", x, E, True, kind) if eight else (_packed(x), None)
    ends = ends.contiguous()
    R = first.shape[0]
    y = torch.empty((R, m), dtype=dtype, device=q.device)
    if R:
        _queue(q.device, "htr_product", q.data_ptr(), _CODE[q.dtype], _ptr(s), w.data_ptr(), _ptr(ws), None, ends.data_ptr(), y.data_ptr(), R, m, n, E, _CODE[w.dtype],
               _CODE[dtype])
    return y


def moe_experts_stacked(x, expert_ids, expert_weights, gate_up, down):
    """ops.moe_experts on matrices that are not HTR-W1: y_t = sum_j w_tj Down_e( silu(Gate_e x_t) * Up_e x_t ), e = ids[t, j].

    x [T, H] in bfloat16 or float16; expert_ids [T, top] int32 or int64; expert_weights [T, top]; gate_up [E, 2F, H] (gate rows first) and down
    [E, H, F] of x's type, H and F multiples of 8, or 8-bit pairs of one kind (e4m3: multiples of 128, int8: of 16), to which x and the hidden values are rounded as well.
    Sums are as in the products, those of gate and up in e4m3 float32 throughout with up to some tens of rows to an expert (an e4m3 rounding follows them);
    the hidden values are rounded to x's type, e4m3 or int8 in between, y [T, H] to x's type.  A token with an expert number out of range
    becomes NaN."""
    eight = _pair(gate_up) and _pair(down)
    path = _fast(x)
    if path is not None:
        (gu, gus), (dn, dns) = (gate_up, down) if eight else ((gate_up, None), (down, None))
        y = path[0].moe_stacked(x, expert_ids, expert_weights, gu, gus, dn, dns, path[1])
        if y is not None:
            if type(y) is int:
                _native.check(y)
            return y
    if x.dim() != 2 or x.dtype not in _HALVES:
        raise RuntimeError("moe_experts_stacked wants x [T, H] in bfloat16 or float16")
    if eight:
        kind = I8 if gate_up[0].dtype is I8 else E4M3
        _check_matrix("moe_experts_stacked", gate_up[0], gate_up[1], 3, kind)
        _check_matrix("moe_experts_stacked", down[0], down[1], 3, kind)
        (gu, gus), (dn, dns) = gate_up, down
    else:
        gu, gus, dn, dns = gate_up, None, down, None
        if _pair(gu) or _pair(dn) or gu.dtype != x.dtype or dn.dtype != x.dtype or gu.dim() != 3 or dn.dim() != 3:
            raise RuntimeError("moe_experts_stacked: gate_up [E, 2F, H] and down [E, H, F] in x's type, or both in 8 bits")
        if not all(w.is_contiguous() and w.data_ptr() % 16 == 0 for w in (gu, dn)):
            raise RuntimeError("moe_experts_stacked: weights must be contiguous, on a 16-byte boundary")
    T, H = x.shape
    E, F = dn.shape[0], dn.shape[2]
    unit = _UNIT[kind] if eight else 8
    if gu.shape != (E, 2 * F, H) or dn.shape[1] != H or E < 1 or F < 1 or H < 1 or H % unit or F % unit:
        raise RuntimeError(f"moe_experts_stacked: gate_up [E, 2F, H] and down [E, H, F], H and F multiples of {unit}")
    if expert_ids.dim() != 2 or expert_ids.shape[0] != T or expert_ids.shape != expert_weights.shape or expert_ids.dtype not in (torch.int32, torch.int64):
        raise RuntimeError("moe_experts_stacked: expert_ids int32 or int64 [T, top], expert_weights [T, top]")
    _on_one_gpu("moe_experts_stacked", x, gu, gus, dn, dns, expert_ids, expert_weights)
    _refuse_derivatives("moe_experts_stacked", x, expert_weights, gu, gus, dn, dns)
    top = expert_ids.shape[1]
    if T == 0 or top == 0:
        return torch.zeros((T, H), dtype=x.dtype, device=x.device)
    x, ids, wt = _packed(x), expert_ids.contiguous(), expert_weights.to(torch.float32).contiguous()
    need = _native.lib().htr_moe_stacked_scratch_bytes(T, top, E, H, F, _CODE[gu.dtype])
    if need == 0:
        raise RuntimeError("moe_experts_stacked: more tokens, slots, experts or columns than a call takes")
    scratch = torch.empty(need, dtype=torch.uint8, device=x.device)
    y = torch.empty((T, H), dtype=x.dtype, device=x.device)
    _queue(x.device, "htr_moe_stacked", x.data_ptr(), _CODE[x.dtype], ids.data_ptr(), int(ids.dtype == torch.int64), wt.data_ptr(), T, top,
           gu.data_ptr(), _ptr(gus), dn.data_ptr(), _ptr(dns), E, H, F, _CODE[gu.dtype], y.data_ptr(), scratch.data_ptr(), need)
    return y


def route_experts(logits, top, scores="softmax", bias=None, groups=1, top_groups=1, group_best=1, renormalize=True, scale=1.0):
    """(ids int32 [..., top], weights float32 [..., top]): each token's experts from a router's logits [..., E], for moe_experts and moe_experts_stacked.

    Scores are the softmax of the logits, or with scores="sigmoid" their sigmoid; the experts come in descending order of score + bias (bias [E]: what balances
    the experts' load, no part of the weights), without a bias of their logits, ties to the lowest number.  With groups, E / groups consecutive experts each, only
    those of the best top_groups groups compete; a group is as good as its best expert, or with group_best=2 the sum of its two best scores + bias.  Weights are
    the scores, divided by their sum with renormalize, times scale.  Logits bfloat16, float16 or float32; scores are 64 bits.
    A logit (or bias) of -inf masks its expert, which comes behind every other, with weight 0; a group is then as good as the experts it has left, and comes behind all others
    without any; a token without any other expert gets weights 0.  NaN ranks first, with weight NaN.
    E up to 1024, groups and top up to 64."""
    path = _fast(logits)
    if path is not None:
        y = path[0].route(logits, top, scores, bias, groups, top_groups, group_best, renormalize, scale, path[1])
        if y is not None:
            return y
    if logits.dim() < 1 or logits.dtype not in _FLOATS or not 1 <= logits.shape[-1] <= 1024:
        raise RuntimeError("route_experts wants logits [..., E] in bfloat16, float16 or float32, E up to 1024")
    E = logits.shape[-1]
    if scores not in ("softmax", "sigmoid"):
        raise RuntimeError('route_experts: scores are "softmax" or "sigmoid"')
    if not 1 <= groups <= 64 or E % groups or not 1 <= top_groups <= groups or group_best not in (1, 2):
        raise RuntimeError("route_experts: groups up to 64 that divide E, top_groups of them, group_best 1 or 2")
    if not 1 <= top <= min(64, E // groups * top_groups):
        raise RuntimeError("route_experts: top is at least 1, at most 64 and at most the experts of top_groups groups")
    if bias is not None and (bias.shape != (E,) or bias.dtype not in _FLOATS):
        raise RuntimeError("route_experts: the bias must be [E] in bfloat16, float16 or float32")
    _on_one_gpu("route_experts", logits, bias)
    _refuse_derivatives("route_experts", logits, bias)
    x, stride = _rows(logits)
    bias = None if bias is None else bias.to(torch.float32).contiguous()
    ids = torch.empty(logits.shape[:-1] + (top,), dtype=torch.int32, device=logits.device)
    weights = torch.empty(ids.shape, dtype=torch.float32, device=logits.device)
    if logits.numel():
        _queue(logits.device, "htr_route", x.data_ptr(), stride, _CODE[logits.dtype], x.shape[0], E, top, int(scores == "sigmoid"), _ptr(bias), groups, top_groups, group_best,
               int(bool(renormalize)), scale, ids.data_ptr(), weights.data_ptr())
    return ids, weights
