"""Calls of the operators around the packed linears that their descriptions do not allow, and are refused as what they are."""
import pytest
import torch

from htr_amd import ops

BF16, E4M3 = torch.bfloat16, torch.float8_e4m3fn


def incomplete_pairs(device):
    x, w = torch.zeros(2, 128, dtype=BF16, device=device), torch.zeros(1, 256, 128, dtype=BF16, device=device)
    q, s = torch.zeros(256, 128, device=device).to(E4M3), torch.ones(2, 1, device=device)
    ends, ids, wt = torch.ones(1, dtype=torch.int32, device=device), torch.zeros(2, 1, dtype=torch.int64, device=device), torch.ones(2, 1, device=device)
    down = torch.zeros(1, 128, 128, dtype=BF16, device=device)
    return [lambda: ops.linear_fp8((x, None), q, s), lambda: ops.linear_fp8([x, None], q, s), lambda: ops.linear_fp8((q, None), q, s), lambda: ops.linear_fp8((x, x, x), q, s),
            lambda: ops.linear_fp8(x, q, None), lambda: ops.linear_fp8(x, None, s), lambda: ops.grouped_mm((x, None), w, ends), lambda: ops.grouped_mm(x, (w, None), ends),
            lambda: ops.grouped_mm((None, s), w, ends), lambda: ops.moe_experts_stacked(x, ids, wt, (w, None), (down, None)),
            lambda: ops.moe_experts_stacked(x, ids, wt, (w, None), down)]


def test_incomplete_pairs_are_refused():
    for k, call in enumerate(incomplete_pairs("cpu")):
        with pytest.raises(RuntimeError, match=r"pair|8-bit weight"):
            call()
            pytest.fail(f"call {k} was taken")


@pytest.mark.gpu
def test_incomplete_pairs_are_refused_on_a_gpu():
    for k, call in enumerate(incomplete_pairs("cuda")):
        with pytest.raises(RuntimeError, match=r"pair|8-bit weight"):
            call()
            pytest.fail(f"call {k} was taken")
