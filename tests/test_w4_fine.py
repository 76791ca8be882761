"""Refusals and sizes of the calls that products of many records per expert need; no GPU."""

import ctypes

import pytest

from moe_inference_verify_microbench_b200 import _native

P = ctypes.c_void_p(4096)  # stand-in address, never dereferenced
ODD = ctypes.c_void_p(4100)


def bank(E=16, H=256, I=128, group=64, zeros=_native.W4_FINE, f=(4096, 4096, 4096, 4096)):
    return ctypes.byref(_native.W4BankStruct(4096, 4096, 4096, 4096, E, H, I, group, zeros, *f))


def test_pack_fine_is_refused_on_the_host():
    pack = _native.load().moe_w4_pack_fine

    def call(s0=P, z0=None, s1=None, z1=None, E=2, N=64, K=128, group=64, f=P, r=P):
        return pack(s0, z0, s1, z1, E, N, K, group, f, r, None)

    assert call(s0=None) == -1
    assert call(f=None) == -1
    assert call(r=None) == -1
    assert call(f=ODD) == -1
    assert call(r=ODD) == -1
    assert call(z1=P) == -1
    assert call(s1=P, z0=P) == -1
    assert call(s1=P, z1=P) == -1
    assert call(E=0) == -1
    assert call(E=1025) == -2
    assert call(group=16) == -2
    assert call(K=96) == -2
    assert call(K=8256) == -2
    assert call(N=40) == -2


@pytest.mark.parametrize("missing", range(4))
def test_bank_has_all_four_or_none(missing):
    """A bank that says it has the fine scales has to have all of them."""
    lib = _native.load()
    f = [4096] * 4
    f[missing] = None
    assert lib.moe_w4_sorted_forward(P, 4, P, bank(f=f), P, 1 << 40, P, None, None) == -1
    f[missing] = 4100
    assert lib.moe_w4_sorted_forward(P, 4, P, bank(f=f), P, 1 << 40, P, None, None) == -1
    # without the flag they are not read: only the workspace is missing here
    assert lib.moe_w4_sorted_forward(P, 4, P, bank(zeros=1, f=f), P, 0, P, None, None) == -5


def test_grouped_calls_with_a_workspace():
    lib = _native.load()
    n13, n2 = (lib.moe_w4_grouped_workspace_bytes(300, c) for c in (256, 128))
    assert n13 >= 300 * 256 * 2 + 300 * 4 and n2 >= 300 * 128 * 2 + 300 * 4
    assert lib.moe_w4_grouped_workspace_bytes(-1, 256) == 0
    assert lib.moe_w4_grouped_workspace_bytes(4, 0) == 0
    w13, w2 = lib.moe_grouped_w13_swiglu_w4_ex, lib.moe_grouped_w2_w4_ex

    def up(b=bank(), src=P, ws=P, n=n13, h=P):
        return w13(src, 300, None, 1, 300, P, P, 3, b, h, ws, n, None, None)

    def down(b=bank(), h=P, ws=P, n=n2, out=P):
        return w2(h, 300, P, P, 3, b, None, None, out, 300, ws, n, None, None)

    for call, need in ((up, n13), (down, n2)):
        assert call(b=None) == -1
        assert call(n=need - 1) == -5
        assert call(ws=ODD) == -1
        assert call(b=bank(group=48)) == -2
    assert up(src=None) == up(h=None) == down(h=None) == down(out=None) == -1


def test_workspaces_hold_the_activations_of_many_records():
    lib = _native.load()
    plain, fine = bank(128, 2048, 768, 128, zeros=0), bank(128, 2048, 768, 128)
    for query, many in ((lib.moe_w4_experts_workspace_bytes, (8192, 8)),
                        (lib.moe_w4_layer_workspace_bytes, (8192, 8))):
        assert query(16, 8, fine) == query(16, 8, plain)  # one record per expert
        T, k = many
        assert query(T, k, fine) >= query(T, k, plain) + T * 2048 * 2 + T * k * 768 * 2
    assert lib.moe_w4_sorted_workspace_bytes(100, fine) == lib.moe_w4_sorted_workspace_bytes(100, plain)
    assert (lib.moe_w4_sorted_workspace_bytes(6000, fine)
            >= lib.moe_w4_sorted_workspace_bytes(6000, plain) + 6000 * (2048 * 2 + 768 * 2))
