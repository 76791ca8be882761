"""Host-side checks of the modules on 4-bit experts and of the block with norms after
its branches; no GPU is needed."""

import ctypes

import pytest
import torch

from moe_inference_verify_microbench_b200 import PermutedSparseMoE, _native, ops, quantize_w4
from moe_inference_verify_microbench_b200.hybrid import HybridBlock, RMSNorm

P = ctypes.c_void_p(4096)  # stand-in address, never dereferenced


def test_module_options_are_refused():
    with pytest.raises(ValueError, match="expert_weights"):
        PermutedSparseMoE(64, 64, 16, 2, expert_weights="int4")
    with pytest.raises(ValueError, match="index_add"):
        PermutedSparseMoE(64, 64, 16, 2, expert_weights="w4", group_size=64, index_add="atomic")
    with pytest.raises(ValueError, match="decode_weights"):
        PermutedSparseMoE(64, 64, 16, 2, expert_weights="w4", group_size=64, decode_weights=True)
    for H, I, group in ((64, 64, 48), (96, 64, 64), (64, 96, 64), (64, 64, 128)):
        with pytest.raises(ValueError, match="group_size"):
            PermutedSparseMoE(H, I, 16, 2, expert_weights="w4", group_size=group)
    mod = PermutedSparseMoE(64, 64, 16, 2)  # the default has no such bank and no such checks
    assert mod.expert_weights == "bf16" and mod._w4 is None


def test_ranges_beyond_the_scales_are_refused():
    top = torch.finfo(torch.float32).max
    w = torch.zeros(2, 64)
    w[0, 0], w[0, 1] = top, -top
    with pytest.raises(ValueError, match="range"):
        quantize_w4(w, 64, symmetric=False)


def block(**options):
    return HybridBlock(64, 64, 2, 2, 32, 4, 2, 1, 0, None, 1, 0, None, **options)


def test_block_options_are_refused():
    with pytest.raises(ValueError, match="post_norm"):
        block(gate_act="tanh")
    with pytest.raises(ValueError, match="post_norm"):
        block(residual_scale=0.5)
    with pytest.raises(ValueError, match="gate_act"):
        block(post_norm=True, gate_act="relu")
    plain = block()
    assert not any("post_norm" in n or n.endswith("_gate") for n, _ in plain.named_parameters()
                   if not n.startswith("moe.experts"))
    x = torch.zeros(1, 2, 64)
    with pytest.raises(ValueError, match="eps"):
        plain(x, next_norm=RMSNorm(64, eps=1e-5))
    with pytest.raises(ValueError, match="normed"):
        plain(x, normed=torch.zeros(1, 3, 64))


def test_block_loads_its_extra_weights():
    def load(blk, **extra):
        z = lambda *s: torch.zeros(*s)
        w = [z(64, 64)] * 4
        blk.weight_loader(z(64), z(64, 64), z(64, 64), z(64, 64), z(64, 64), z(64), z(4, 64), w, w,
                          w, **extra)

    full = block(post_norm=True, gate_act="sigmoid")
    load(full, attn_post_norm_weight=torch.full((64,), 2.0), moe_gate=torch.full((64,), 3.0))
    assert bool((full.attn_post_norm.weight == 2.0).all()) and bool((full.moe_gate == 3.0).all())
    assert bool((full.moe_post_norm.weight == 1.0).all()) and bool((full.attn_gate == 1.0).all())
    with pytest.raises(ValueError, match="no attn_gate"):
        load(block(post_norm=True), attn_gate=torch.ones(64))
    with pytest.raises(ValueError, match="no moe_post_norm"):
        load(block(), moe_post_norm_weight=torch.ones(64))


def test_sorted_rows_are_refused_on_the_host():
    lib = _native.load()

    def bank(H=256, group=64):
        return ctypes.byref(_native.W4BankStruct(4096, 4096, 4096, 4096, 16, H, 128, group, 0))

    def call(x=P, M=40, off=P, b=None, ws=P, n=1 << 40, y=P):
        return lib.moe_w4_sorted_forward(x, M, off, b if b is not None else bank(), ws, n, y, None,
                                         None)

    assert call(M=-1) == -1
    assert call(x=None) == -1
    assert call(off=None) == -1
    assert call(y=None) == -1
    assert call(y=ctypes.c_void_p(4098)) == -1
    assert call(ws=None) == -1
    assert call(n=64) == -5
    assert call(b=bank(H=96)) == -2
    assert call(b=bank(group=40)) == -2
    assert call(M=0, x=None, y=None, ws=None, n=0) == 0
    assert lib.moe_w4_sorted_forward(P, 4, P, None, P, 1 << 30, P, None, None) == -1
    assert lib.moe_w4_sorted_workspace_bytes(40, bank()) > 40 * 128 * 2
    assert lib.moe_w4_sorted_workspace_bytes(-1, bank()) == 0
    assert lib.moe_w4_sorted_workspace_bytes(40, None) == 0


def test_layer_takes_the_routers_numbers_of_experts():
    lib = _native.load()
    for E, want in ((24, -2), (8, -2), (272, -2), (16, -5)):  # 16: only the workspace is missing
        b = ctypes.byref(_native.W4BankStruct(4096, 4096, 4096, 4096, E, 256, 128, 64, 0))
        for T in (1, 12, 300):
            assert lib.moe_w4_layer_forward(P, P, None, b, T, 2, 1, P, 0, P, None, None) == want


def test_tile_tables_are_read_by_sixteen_bytes():
    lib = _native.load()
    b = ctypes.byref(_native.W4BankStruct(4096, 4096, 4096, 4096, 16, 256, 128, 64, 0))
    odd = ctypes.c_void_p(4100)
    assert lib.moe_grouped_w13_swiglu_w4(P, 5, None, 1, 5, odd, P, 3, b, P, None, None) == -1
    assert lib.moe_grouped_w2_w4(P, 5, odd, P, 3, b, None, None, P, 5, None, None) == -1
    assert lib.moe_grouped_w13_swiglu_w4(P, 0, P, 1, 5, P, P, 3, b, P, None, None) == -1  # no rows


def test_gate_activations():
    assert [ops.check_gate_act(a) for a in ("none", "sigmoid", "tanh")] == [0, 1, 2]
