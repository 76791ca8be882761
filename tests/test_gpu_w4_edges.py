"""The 4-bit experts and the block norm at the calls where they could go wrong: weights
written after a forward, rows that no expert owns, tensors in place, rows and forms
beside one another."""

import pytest
import torch

import w4_reference as ref
from moe_inference_verify_microbench_b200 import PermutedSparseMoE, ops, quantize_w4
from test_gpu_w4 import close, rms_close, rows
from test_gpu_w4_layers import module

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------ weights written later


def test_module_after_load_state_dict(cuda):
    """Forward, load, forward: the second answers for the weights that were loaded."""
    H, E, k = 256, 16, 4
    mod = module(cuda, H=H, group_size=64)
    torch.manual_seed(6)
    other = PermutedSparseMoE(H, 128, E, k).to(device=cuda, dtype=torch.bfloat16)
    x = rows(6, H, 3, cuda)
    with torch.no_grad():
        first = mod(x)
        mod.load_state_dict(other.state_dict())
        second = mod(x)
        assert not torch.equal(first, second)
        ids, w, _ = ops.router_topk(x, other.gate.weight, k)
        parts = [quantize_w4(t, 64) for t in other.pack()]
        want, bound = ref.experts(parts, x, ids, w)
        close(second, want, bound)
        rms_close(second, want, "y", False)
        mod.experts[3].down_proj.weight.zero_()
        parts[2][0][3] = 8  # codes of zero
        close(mod(x), *ref.experts(parts, x, ids, w))
    ops.check_status(cuda)


def test_decode_weights_after_load_state_dict(cuda):
    H, I, E, k = 256, 128, 16, 4
    make = lambda **o: PermutedSparseMoE(H, I, E, k, **o).to(device=cuda, dtype=torch.bfloat16)
    mod, other = make(decode_weights=True), make(decode_weights=True)
    x = rows(2, H, 3, cuda)
    with torch.no_grad():
        mod(x)
        mod.load_state_dict(other.state_dict())
        assert torch.equal(mod(x), other(x))
    ops.check_status(cuda)
