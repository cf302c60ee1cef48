"""The operators around the packed linears: the norm in front of them, and linears and routed experts that a checkpoint leaves out of HTR-W1.

    y, h = ops.rms_norm(x, weight, residual=h)                           # 16-bit result, for ops.linear
    xq, h = ops.rms_norm(x, weight, residual=h, quantize=True)           # (e4m3 values, scales), for the two below
    y = ops.linear_fp8(xq, qweight, scales)                              # weight in e4m3 with a scale for each 128x128 block
    y = ops.grouped_mm(xs, weights, ends)                                # rows sorted by expert, stacked matrices in 16 or 8 bits
    y = ops.moe_experts_stacked(x, ids, weights, gate_up, down)          # ops.moe_experts on such matrices

The reference leaves these modules to its caller (its plugin returns UnquantizedLinearMethod, htr/vllm_plugin.py:49-69).

8-bit rows are a pair (values float8_e4m3fn [..., n], scales float32 [..., n / 128]), 8-bit matrices a pair (values [.., m, n], scales
[.., ceil(m / 128), n / 128]); a value stands for itself times its block's scale.  The scales made here are powers of two, the least that brings
the block to 448 or below; scales from elsewhere need not be.  Infinities and NaN become NaN.

Norms sum in 64 bits, products of 16-bit values in float32.  Products of e4m3 values are first added eight consecutive
columns at a time, as the matrix instructions do: each eight is off by at most 2^-10 of the largest magnitude in x times that in the matrix (one below 2^-6 of its
scale counts as that).  Everything beyond is float32, the product of a row's scale and a block's as well (below 2^-126 it has fewer bits, beyond float32 it is
infinite).  Results are rounded once.  Nothing here has a derivative, as no packed linear has one in its
activations: a call that torch would differentiate is refused.  Calls only queue kernels on the current stream of x's device, allocate with torch and
may be captured into a graph.
"""
import torch

from . import _native

E4M3 = torch.float8_e4m3fn
_CODE = {torch.bfloat16: _native.BF16, torch.float16: _native.F16, torch.float32: _native.F32, E4M3: _native.E4M3}
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
    (values, scales) of y in e4m3 (n a multiple of 128); with a residual, (that, t): t is the next block's residual."""
    path = _fast(x)
    if path is not None:
        y = path[0].rms_norm(x, weight, eps, residual, quantize, path[1])
        if y is not None:
            return y
    if x.dim() < 1 or x.dtype not in _FLOATS or weight.dtype != x.dtype or weight.shape != x.shape[-1:]:
        raise RuntimeError("rms_norm wants x [..., n] in bfloat16, float16 or float32 and a weight [n] of that type")
    if residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype):
        raise RuntimeError("rms_norm: the residual must have x's shape and type")
    n = x.shape[-1]
    if n < 1 or (quantize and n % 128):
        raise RuntimeError("rms_norm: at least one column, and a multiple of 128 for an 8-bit result")
    _on_one_gpu("rms_norm", x, weight, residual)
    _refuse_derivatives("rms_norm", x, weight, residual)
    x2, xs = _rows(x)
    r2, rs = (None, 0) if residual is None else _rows(residual)
    w = weight.contiguous()
    y = torch.empty(x.shape, dtype=E4M3 if quantize else x.dtype, device=x.device)
    scales = torch.empty(x.shape[:-1] + (n // 128,), dtype=torch.float32, device=x.device) if quantize else None
    total = None if residual is None else torch.empty(x.shape, dtype=x.dtype, device=x.device)
    if x.numel():
        _queue(x.device, "htr_rms_norm", x2.data_ptr(), xs, _ptr(r2), rs, w.data_ptr(), x2.shape[0], n, eps, _CODE[x.dtype], y.data_ptr(),
               _ptr(scales), _ptr(total))
    out = (y, scales) if quantize else y
    return out if residual is None else (out, total)


def _ptr(t):
    return None if t is None else t.data_ptr()


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


def _check_rows(what, x, experts, grouped):
    """x as htr_product takes it with an 8-bit weight: contiguous 8-bit rows (values, scales), to which a tensor is rounded, or few 16-bit rows (x, None)."""
    if not _pair(x):
        n = x.shape[-1]
        if x.dtype in _HALVES and n % 128 == 0 and n and _native.lib().htr_product_rounds(x.numel() // n, experts, int(grouped)):
            return _packed(x), None
        return quantize_fp8(x)
    q, s = x
    if q.dtype != E4M3 or s.dtype != torch.float32 or q.dim() < 1 or s.shape != q.shape[:-1] + (q.shape[-1] // 128,) or q.shape[-1] % 128:
        raise RuntimeError(f"{what}: 8-bit rows are (float8_e4m3fn [..., n], float32 [..., n / 128]), n a multiple of 128")
    return _packed(q), s.contiguous()


def _check_matrix(what, q, s, dims):
    if not isinstance(q, torch.Tensor) or not isinstance(s, torch.Tensor) or q.dtype != E4M3 or s.dtype != torch.float32 or q.dim() != dims or q.shape[-1] % 128 or 0 in q.shape \
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
    y = _product(x, qweight, scales, bias, None, out_dtype)
    if y is not None:
        return y
    _check_matrix("linear_fp8", qweight, scales, 2)
    m, n = qweight.shape
    dtype = _out_dtype("linear_fp8", out_dtype, x, bias)
    first = x[0] if _pair(x) else x
    if first.dim() < 1 or first.shape[-1] != n:
        raise RuntimeError(f"linear_fp8: x has {first.shape[-1] if first.dim() else 0} columns, the weight {n}")
    if bias is not None and (bias.dtype != dtype or bias.shape != (m,)):
        raise RuntimeError("linear_fp8: the bias must be [m] in the result's type")
    _on_one_gpu("linear_fp8", first, qweight, scales, bias, x[1] if _pair(x) else None)
    _refuse_derivatives("linear_fp8", *(x if _pair(x) else (x,)), qweight, scales, bias)
    q, s = _check_rows("linear_fp8", x, 1, False)
    bias = None if bias is None else bias.contiguous()
    y = torch.empty(first.shape[:-1] + (m,), dtype=dtype, device=q.device)
    if y.numel():
        _queue(q.device, "htr_product", q.data_ptr(), _CODE[q.dtype], _ptr(s), qweight.data_ptr(), scales.data_ptr(), _ptr(bias), None, y.data_ptr(), y.numel() // m,
               m, n, 1, _native.E4M3, _CODE[dtype])
    return y


def grouped_mm(x, weight, ends, out_dtype=None):
    """Rows sorted by expert times their expert's matrix: y[r] = W_e x[r] for ends[e - 1] <= r < ends[e] (from 0).

    weight: [E, m, n] in bfloat16 or float16, x [R, n] of the same type, n a multiple of 8; or an 8-bit pair (values [E, m, n], scales), with x in
    8-bit rows or rounded to them.  ends: int32 [E] on the device (the running sum of the experts' row counts); an end below an earlier one counts as
    that one, one beyond R as R; rows from the last end on become zeros.  y [R, m] in x's type (8-bit rows: bfloat16) unless out_dtype says."""
    eight = _pair(weight)
    if ends is not None:
        y = _product(x, weight[0], weight[1], None, ends, out_dtype) if eight else _product(x, weight, None, None, ends, out_dtype)
        if y is not None:
            return y
    first = x[0] if _pair(x) else x
    if eight:
        _check_matrix("grouped_mm", weight[0], weight[1], 3)
        w, ws = weight
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
    q, s = _check_rows("grouped_mm", x, E, True) if eight else (_packed(x), None)
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
    [E, H, F] of x's type, H and F multiples of 8, or 8-bit pairs (multiples of 128), with which x and the hidden values are rounded to e4m3 as well.
    Sums are as in the products, those of gate and up in 8 bits float32 throughout with up to some tens of rows to an expert (an e4m3 rounding follows them);
    the hidden values are rounded to x's type or e4m3 in between, y [T, H] to x's type.  A token with an expert number out of range
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
        _check_matrix("moe_experts_stacked", gate_up[0], gate_up[1], 3)
        _check_matrix("moe_experts_stacked", down[0], down[1], 3)
        (gu, gus), (dn, dns) = gate_up, down
    else:
        gu, gus, dn, dns = gate_up, None, down, None
        if _pair(gu) or _pair(dn) or gu.dtype != x.dtype or dn.dtype != x.dtype or gu.dim() != 3 or dn.dim() != 3:
            raise RuntimeError("moe_experts_stacked: gate_up [E, 2F, H] and down [E, H, F] in x's type, or both in 8 bits")
        if not all(w.is_contiguous() and w.data_ptr() % 16 == 0 for w in (gu, dn)):
            raise RuntimeError("moe_experts_stacked: weights must be contiguous, on a 16-byte boundary")
    T, H = x.shape
    E, F = dn.shape[0], dn.shape[2]
    unit = 128 if eight else 8
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
