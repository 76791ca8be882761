"""The 4-bit experts and the block norm without a GPU: quantisation, refusals and
the sizes the library answers for."""

import ctypes

import pytest
import torch

from moe_inference_verify_microbench_b200 import W4Experts, _native, dequantize_w4, ops, quantize_w4


@pytest.mark.parametrize("symmetric", [True, False])
@pytest.mark.parametrize("group", [32, 64, 128])
def test_quantize_is_nearest(symmetric, group):
    gen = torch.Generator().manual_seed(group)
    w = torch.randn((3, 16, 256), generator=gen) * 0.02
    w[0, 0] = 0.0
    w[1, 1, :group] = 0.5
    codes, scales, zeros = quantize_w4(w, group, symmetric)
    assert codes.dtype == torch.uint8 and int(codes.max()) <= 15
    assert scales.dtype == torch.bfloat16 and scales.shape == (3, 16, 256 // group)
    assert (zeros is None) == symmetric
    back = dequantize_w4(codes, scales, zeros)
    # half a step, and what the scale's rounding to bf16 moves the ends of the range by
    # (15 steps of 2^-8 each); a zero point is itself rounded, by half a step
    step = scales.float().repeat_interleave(group, -1)
    slack = 0.5 + 15 * 2.0 ** -8 + (0.0 if symmetric else 0.5)
    assert ((back - w).abs() <= slack * step + 1e-12).all()
    assert not back[0, 0].any()


def test_quantize_refusals():
    w = torch.zeros((4, 256))
    with pytest.raises(ValueError, match="group_size"):
        quantize_w4(w, 48)
    with pytest.raises(ValueError, match="multiple"):
        quantize_w4(torch.zeros((4, 96)), 64)
    with pytest.raises(TypeError):
        quantize_w4(torch.zeros((4, 64), dtype=torch.int32), 64)
    w[1, 2] = float("nan")
    with pytest.raises(ValueError, match="infinity or a NaN"):
        quantize_w4(w, 64)


def test_cpu_tensors_are_refused():
    c = torch.zeros((2, 64, 64), dtype=torch.uint8)
    s = torch.ones((2, 64, 1), dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="no CPU path"):
        W4Experts.from_codes((c, s, None), (c, s, None), (c, s, None))
    x = torch.zeros((3, 64), dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="no CPU path"):
        ops.block_norm(x, x, torch.ones(64), torch.ones(64), 1e-6)
    with pytest.raises(ValueError, match="no CPU path"):
        ops.experts_w4(x, torch.zeros((3, 2), dtype=torch.int32), torch.zeros((3, 2)), None)


P = ctypes.c_void_p(4096)  # stand-in address, never dereferenced


def bank(E=16, H=256, I=128, group=64, **ptr):
    fields = dict(w13_q=4096, w13_s=4096, w2_q=4096, w2_s=4096)
    fields.update(ptr)
    return ctypes.byref(_native.W4BankStruct(fields["w13_q"], fields["w13_s"], fields["w2_q"],
                                             fields["w2_s"], E, H, I, group, 0))


def layer(b, T=4, k=4, x=P, wr=P, ws=P, ws_bytes=1 << 40, y=P):
    return _native.load().moe_w4_layer_forward(x, wr, None, b, T, k, 1, ws, ws_bytes, y, None, None)


def experts(b, T=4, k=4, E=16, e0=0, x=P, ids=P, w=P, ws=P, ws_bytes=1 << 40, y=P):
    return _native.load().moe_w4_experts_forward(x, ids, w, T, k, E, e0, b, ws, ws_bytes, y, None,
                                                 None)


@pytest.mark.parametrize("call", [layer, experts])
def test_calls_are_refused_on_the_host(call):
    assert call(None) == -1
    assert call(bank(), T=-1) == -1
    assert call(bank(), k=0) == -1
    assert call(bank(), k=9) == -2
    assert call(bank(group=48)) == -2
    assert call(bank(H=96)) == -2
    assert call(bank(I=64, group=128)) == -2
    assert call(bank(H=8256)) == -2
    assert call(bank(w13_q=None)) == -1
    assert call(bank(w2_q=4100)) == -1           # misaligned
    assert call(bank(), x=None) == -1
    assert call(bank(), y=None) == -1
    assert call(bank(), y=ctypes.c_void_p(4098)) == -1
    assert call(bank(), ws=None) == -1
    assert call(bank(), ws_bytes=100) == -5
    assert call(bank(), T=(1 << 31) // 4) == -2  # 2^31 records
    assert call(bank(), T=0, x=None, y=None, ws=None, ws_bytes=0) == 0


def test_experts_range_is_checked():
    assert experts(bank(), E=15) == -1
    assert experts(bank(E=4), E=16, e0=13) == -1
    assert experts(bank(), e0=-1, E=32) == -1
    assert experts(bank(), ids=None) == -1
    assert experts(bank(), T=0, ids=None, w=None) == 0


def test_layer_needs_the_router():
    assert layer(bank(), wr=None) == -1
    assert layer(bank(E=4), k=5) == -1


def test_grouped_calls_are_refused_on_the_host():
    lib = _native.load()
    b = bank()
    w13, w2 = lib.moe_grouped_w13_swiglu_w4, lib.moe_grouped_w2_w4
    assert w13(P, 5, None, 1, 5, P, P, 3, None, P, None, None) == -1
    assert w13(P, 5, None, 0, 5, P, P, 3, b, P, None, None) == -1
    assert w13(None, 5, None, 1, 5, P, P, 3, b, P, None, None) == -1
    assert w13(P, 5, None, 1, 5, None, P, 3, b, P, None, None) == -1
    assert w13(ctypes.c_void_p(4098), 5, None, 1, 5, P, P, 3, b, P, None, None) == -1
    assert w13(None, 0, None, 1, 0, P, P, 3, b, None, None, None) == 0
    assert w2(P, 5, P, P, 3, None, None, None, P, 5, None, None) == -1
    assert w2(P, 5, P, P, 3, b, None, None, None, 5, None, None) == -1
    assert w2(None, 0, P, P, 3, b, None, None, None, 0, None, None) == 0


def test_pack_is_refused_on_the_host():
    pack = _native.load().moe_w4_pack

    def call(c0=P, s0=P, z0=None, c1=None, s1=None, z1=None, E=2, N=64, K=128, group=64, q=P, s=P):
        return pack(c0, s0, z0, c1, s1, z1, E, N, K, group, q, s, None, None)

    assert call(c0=None) == -1
    assert call(c1=P) == -1
    assert call(z1=P) == -1
    assert call(c1=P, s1=P, z0=P) == -1
    assert call(E=0) == -1
    assert call(group=16) == -2
    assert call(K=96) == -2
    assert call(K=8192 + 64) == -2
    assert call(N=40) == -2
    assert call(c0=ctypes.c_void_p(4097)) == -1


def test_block_norm_is_refused_on_the_host():
    f = _native.load().moe_block_norm

    def call(x=P, d=P, post=P, pre=P, gate=None, kind=0, act=0, T=3, H=256, eps=1e-6, h=P, y=P):
        return f(x, d, post, pre, gate, kind, 0, act, 1.0, T, H, eps, h, y, None)

    assert call(x=None) == -1
    assert call(post=None) == -1
    assert call(kind=2) == -1               # a gate without its values
    assert call(kind=4, gate=P) == -1
    assert call(act=3) == -1
    assert call(H=252) == -2
    assert call(H=32776) == -2
    assert call(H=0) == -1
    assert call(eps=float("nan")) == -1
    assert call(T=-1) == -1
    assert call(y=ctypes.c_void_p(4100)) == -1
    assert call(gate=ctypes.c_void_p(4104), kind=2) == -1
    assert call(T=0, x=None, d=None, h=None, y=None) == 0


def test_workspace_queries():
    lib = _native.load()
    b = bank(E=128, H=2048, I=768, group=128)
    n = lib.moe_w4_experts_workspace_bytes(256, 8, b)
    assert n >= 256 * 8 * (768 + 2048) * 2
    assert lib.moe_w4_layer_workspace_bytes(256, 8, b) >= n + 256 * 8 * 8
    assert lib.moe_w4_experts_workspace_bytes(-1, 8, b) == 0
    assert lib.moe_w4_layer_workspace_bytes((1 << 31) // 8, 8, b) == 0
    assert lib.moe_w4_layer_workspace_bytes(4, 8, None) == 0
