"""The 4-bit experts and the block norm at the calls where they could go wrong: weights
written after a forward, rows that no expert owns, tensors in place, rows and forms
beside one another."""

import copy
import os
import subprocess
import sys

import pytest
import torch

import test_gpu_w4 as w4
import w4_reference as ref
from moe_inference_verify_microbench_b200 import (PermutedSparseMoE, W4Experts,
                                                  fused_moe_forward_w4, ops, quantize_w4)
from test_gpu_w4 import bank_of, close, rms_close, rows
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


@pytest.mark.parametrize("options", [{"expert_weights": "w4", "group_size": 64},
                                     {"decode_weights": True}, {}])
def test_module_under_inference_mode(cuda, options):
    """First run, writes and further runs under inference mode."""
    H = 256
    torch.manual_seed(5)
    make = lambda: PermutedSparseMoE(H, 128, 16, 4, **options).to(device=cuda, dtype=torch.bfloat16)
    mod, other = make(), make()
    x = rows(3, H, 3, cuda)
    with torch.inference_mode():
        mod(x)
        mod.load_state_dict(other.state_dict())
        assert torch.equal(mod(x), other(x))
        mod.experts[2].down_proj.weight.zero_()
        other.pack()[2][2].zero_()
        assert torch.equal(mod(x), other(x))
    ops.check_status(cuda)


def test_copied_module_and_bank(cuda):
    mod = module(cuda, group_size=64)
    x = rows(3, 256, 3, cuda)
    with torch.no_grad():
        y = mod(x)
        bank = copy.deepcopy(mod.experts_4bit())
        assert torch.equal(ops.moe_layer_w4(x, mod.gate.weight, bank, 4), y)
        twin = copy.deepcopy(mod)
        assert torch.equal(twin(x), y)
        twin.experts[0].up_proj.weight.zero_()
        twin.gate.weight.zero_()  # experts 0..3 of every token
        mod.gate.weight.zero_()
        assert not torch.equal(twin(x), mod(x))
    ops.check_status(cuda)


@pytest.mark.parametrize("options", [{"expert_weights": "w4", "group_size": 64},
                                     {"expert_weights": "w4", "group_size": 32, "symmetric": False},
                                     {"decode_weights": True}])
def test_captured_forward_follows_the_weights(cuda, options):
    """A copy that is made again takes the place of the old one in memory, so a captured
    forward reads the new weights, not memory that was freed."""
    H = 256
    torch.manual_seed(5)
    mod = PermutedSparseMoE(H, 128, 16, 4, **options).to(device=cuda, dtype=torch.bfloat16)
    x = rows(3, H, 3, cuda)

    def places():
        if "decode_weights" in options:
            return [mod.down_weights_transposed().data_ptr()]
        bank = mod.experts_4bit()
        return [t.data_ptr() for t in (*bank.w13, *bank.w2)]

    with torch.no_grad():
        mod(x)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = mod(x)
        was = places()
        for _ in range(2):
            state = {n: torch.randn_like(t) * 0.05 for n, t in mod.state_dict().items()}
            mod.load_state_dict(state)
            want = mod(x).clone()
            assert places() == was  # before the replay: it must not read anything else
            torch.cuda.empty_cache()
            graph.replay()
            assert torch.equal(out, want)
        with torch.inference_mode():
            mod.experts[0].down_proj.weight.mul_(3.0)
            want = mod(x).clone()
        mod.experts[0].down_proj.weight.mul_(1.0)
        assert places() == was
        graph.replay()
        assert torch.equal(out, want)
    ops.check_status(cuda)


@pytest.mark.parametrize("run_before", [True, False])
def test_transposed_weights_of_a_capture_are_not_kept(cuda, run_before):
    """Weights written before a capture: what the capture only records, an eager forward does
    not take for done."""
    H = 256
    torch.manual_seed(5)
    make = lambda: PermutedSparseMoE(H, 128, 16, 4, decode_weights=True).to(device=cuda, dtype=torch.bfloat16)
    mod, other = make(), make()
    x = rows(2, H, 3, cuda)
    with torch.no_grad():
        want = other(x)
        mod.pack()
        if run_before:
            mod(x)
        mod.load_state_dict(other.state_dict())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = mod(x)
        assert torch.equal(mod(x), want)
        graph.replay()
        assert torch.equal(out, want)
    ops.check_status(cuda)


# ------------------------------------------------------------------ rows of no expert


@pytest.mark.parametrize("counts", [[0, 3, 1, 9], [128, 0, 60, 129], [0, 0, 0, 0]])
@pytest.mark.parametrize("lead,extra", [(1, 0), (5, 2), (300, 0), (130, 170)])
def test_rows_before_the_first_expert(cuda, counts, lead, extra):
    """Offsets that start above 0: the rows before them are zero, as those past the last
    are, whatever stood in the output (both forms of the product)."""
    E, H, I = 4, 256, 192
    p = ref.parts(E, H, I, 64, True, device=cuda)
    bank = bank_of(p)
    off = (torch.tensor([0] + counts).cumsum(0) + lead).to(cuda)
    M = int(off[-1]) + extra
    x = rows(M, H, 3, cuda)
    out = torch.full((M, H), 7.0, dtype=torch.bfloat16, device=cuda)
    y = ops.sorted_experts_w4(x, off, bank, out=out)
    ops.check_status(cuda)
    assert not bool(y[:lead].any()) and not bool(y[int(off[-1]):].any())
    owner = torch.full((M, 1), -1, device=cuda)
    owner[lead:int(off[-1]), 0] = torch.repeat_interleave(torch.arange(E, device=cuda), off.diff())
    want, bound = ref.experts(p, x, owner, torch.ones((M, 1), device=cuda))
    close(y, want, bound)
    assert torch.equal(y, fused_moe_forward_w4(x, off, bank))


@pytest.mark.parametrize("M", [12, 400])
@pytest.mark.parametrize("offsets", [[0, 5, 3, 9, 10], [-2, 0, 3, 6, 10], [0, 3, 6, 8, "M+1"],
                                     [4, 3, 2, 1, 0], [0, 5, 5, 1 << 40, 1 << 41]])
def test_bad_offsets_are_reported_and_give_zeros(cuda, M, offsets):
    E, H, I = 4, 256, 192
    bank = bank_of(ref.parts(E, H, I, 64, False, device=cuda))
    off = torch.tensor([M + 1 if o == "M+1" else o for o in offsets], device=cuda)
    out = torch.full((M, H), 7.0, dtype=torch.bfloat16, device=cuda)
    ops.sorted_experts_w4(rows(M, H, 3, cuda), off, bank, out=out)
    with pytest.raises(ops.MoEKernelError, match="row index"):
        ops.check_status(cuda)
    assert not bool(out.any())


@pytest.mark.parametrize("M,offsets,want", [
    (200, [0, 2 ** 31 - 1, 0, 100], [[2, 0, 100]]),
    (200, [0, 100, 2 ** 31 - 1, 50, 179], [[0, 0, 100], [3, 50, 178], [3, 178, 179]]),
    (0, [0, 7, 7, 7], [[0, 0, 7]]),
    (100, [0, 2 ** 31 - 1] + [0, 2 ** 31 - 1] * 300, [])])
def test_tile_table_of_experts_with_too_many_rows(cuda, M, offsets, want):
    """An expert with more rows than the table has room for is left out and reported; the
    entries of the others stand at their places in the table, and nothing around it changes."""
    E = len(offsets) - 1
    lib = ops._native.load()
    mt = int(lib.moe_max_tiles(M, E))
    mem = torch.full((mt + 64, 4), -7, dtype=torch.int32, device=cuda)
    num = torch.full((1,), -7, dtype=torch.int32, device=cuda)
    off = torch.tensor(offsets, device=cuda)
    tiles = mem[32:]
    rc = lib.moe_tiles_from_offsets(ops._p(off), E, ops._p(tiles), mt, ops._p(num),
                                    ops._p(ops.status_word(cuda)), ops._stream(cuda))
    assert rc == 0
    if len(want) < E and M:
        with pytest.raises(ops.MoEKernelError, match="row index"):
            ops.check_status(cuda)
    n = int(num)
    assert tiles[:n, :3].tolist() == want
    assert bool((mem[:32] == -7).all()) and bool((tiles[n:] == -7).all())


# ------------------------------------------------------------------ block norm


def norm_call(x, delta, post, pre, gate, kind, h, y, scale=0.7, act=2):
    """The C entry point with outputs of the caller's choice."""
    p = ops._p
    T, H = x.shape
    rc = ops._native.load().moe_block_norm(
        p(x), p(delta), p(post), p(pre), p(gate), kind, int(gate.dtype is torch.float32), act,
        scale, T, H, 1e-6, p(h), p(y), ops._stream(x.device))
    assert rc == 0


# rows whose ends share cache lines (264, 1032) and whole ones; a CTA for a row with 1, 2 and
# 4 vectors a thread, and rows streamed through shared memory with every number of them
@pytest.mark.parametrize("T,H", [(3, 264), (700, 264), (1500, 2056), (1100, 8192), (5, 16392),
                                 (8200, 1032), (2100, 4104), (2100, 5120), (2100, 8192)])
@pytest.mark.parametrize("kind", [2, 3])
def test_block_norm_in_place(cuda, T, H, kind):
    """h written over x and y over delta, either or both: the same as into memory of their
    own, in every form of the kernel."""
    gen = torch.Generator().manual_seed(T + H)
    x = (torch.randn((T, H), generator=gen) * 2).bfloat16().to(cuda)
    d = (torch.randn((T, H), generator=gen) * 0.5).bfloat16().to(cuda)
    post, pre = ((torch.randn(H, generator=gen) * 0.2 + 1).to(cuda) for _ in range(2))
    g = torch.randn((T, H) if kind == 3 else (H,), generator=gen).bfloat16().to(cuda)
    h, y = torch.empty_like(x), torch.empty_like(x)
    norm_call(x, d, post, pre, g, kind, h, y)
    wh, wy, bh, by = ref.block_norm(x, d, post, pre, 1e-6, g, "tanh", 0.7)
    close(h, wh, bh, "h")
    close(y, wy, by, "y")
    for over_x, over_d in ((True, False), (False, True), (True, True)):
        a, b = x.clone(), d.clone()
        h2 = a if over_x else torch.empty_like(x)
        y2 = b if over_d else torch.empty_like(x)
        norm_call(a, b, post, pre, g, kind, h2, y2)
        assert torch.equal(h2, h) and torch.equal(y2, y), (over_x, over_d)


@pytest.mark.parametrize("T", [1, 8192])
def test_block_norm_is_given_the_status_word(cuda, T, monkeypatch):
    """A wait that runs out in it is reported where ``check_status`` reads it."""
    seen = []
    lib = ops._native_lib()

    class Spy:
        def __getattr__(self, name):
            def call(*args):
                seen.append((name, args))
                return getattr(lib, name)(*args)
            return call

    monkeypatch.setattr(ops, "_lib", Spy())
    x, one = rows(T, 2048, 1, cuda), torch.ones(2048, device=cuda)
    ops.block_norm(x, x, one, one, 1e-6)
    (name, args), = seen
    assert name == "moe_block_norm_ex" and args[-2] == ops.status_word(cuda).data_ptr()
    assert "rows of the block norm" in ops._native.error_string(0x107)


# ------------------------------------------------------------------ the forms of the products


# groups of 128 with zero points: one to four shares of a warp, odd numbers of groups, more
# row tiles than a unit of the tensor-memory form holds
@pytest.mark.parametrize("E,H,I", [(3, 128, 128), (4, 384, 256), (6, 2048, 768), (3, 1280, 384),
                                   (2, 8192, 128), (2, 256, 4096)])
@pytest.mark.parametrize("shift", [1, 6, 10, 100, 104, 106])
def test_group_128_with_zero_points(cuda, E, H, I, shift):
    w4.test_grouped_products(cuda, E, H, I, 128, True, shift)


@pytest.mark.parametrize("E,H,I,k,T,bias,norm", [
    (16, 128, 128, 4, 1, False, True), (16, 2048, 768, 8, 8, True, False),
    (128, 2048, 768, 8, 1, False, True), (32, 1280, 384, 4, 16, False, False),
    (16, 4096, 128, 2, 3, False, True), (16, 256, 1408, 4, 5, True, True),
    (16, 512, 256, 4, 33, False, True), (16, 256, 128, 2, 500, True, True)])
def test_layer_of_group_128_with_zero_points(cuda, E, H, I, k, T, bias, norm):
    w4.test_layer(cuda, E, H, I, 128, True, k, T, bias, norm)


@pytest.mark.parametrize("E,H,I,group,zeros,k,T", [
    (16, 256, 128, 64, False, 4, 16), (32, 4096, 128, 128, True, 2, 2), (48, 512, 384, 32, True, 8, 8),
    (128, 2048, 768, 128, False, 8, 7), (16, 2560, 64, 64, True, 4, 13)])
def test_tokens_alone_and_in_a_batch(cuda, E, H, I, group, zeros, k, T):
    """The one-kernel layer gives a token the same row whatever comes with it."""
    p = ref.parts(E, H, I, group, zeros, seed=T, device=cuda)
    bank = bank_of(p)
    x = rows(T, H, 3, cuda)
    router = (torch.randn((E, H), generator=torch.Generator().manual_seed(T)) * 1.8
              * H ** -0.5).bfloat16().to(cuda)
    y = ops.moe_layer_w4(x, router, bank, k)
    for i in range(T):
        assert torch.equal(ops.moe_layer_w4(x[i:i + 1].contiguous(), router, bank, k), y[i:i + 1])
    ops.check_status(cuda)


@pytest.mark.parametrize("group,zeros", [(64, False), (32, True), (128, True)])
@pytest.mark.parametrize("T", [40, 301])
def test_non_finite_rows_in_the_tensor_memory_form(cuda, group, zeros, T):
    """Infinities and NaN stay in their token also where they stand in the first row of an
    expert's tile, which fills the columns past the last record."""
    E, H, I, k = 4, 256, 128, 2
    assert T * k // E >= ref.TC_RECORDS
    p = ref.parts(E, H, I, group, zeros, device=cuda)
    bank = bank_of(p)
    gen = torch.Generator().manual_seed(1)
    ids = torch.rand((T, E), generator=gen).argsort(1)[:, :k].int().contiguous().to(cuda)
    w = torch.rand((T, k), generator=gen).to(cuda)
    x = rows(T, H, 2, cuda)
    clean = ops.experts_w4(x, ids, w, bank)
    bad = {0: float("nan"), 1: float("inf"), 5: float("-inf"), T - 1: float("nan")}
    for n, v in bad.items():
        x[n, (17 * n) % H] = v
    y = ops.experts_w4(x, ids, w, bank)
    ops.check_status(cuda)
    keep = torch.ones(T, dtype=torch.bool, device=cuda)
    keep[list(bad)] = False
    assert bool(torch.isfinite(clean.float()).all()) and torch.equal(y[keep], clean[keep])
    assert not bool(torch.isfinite(y[~keep].float()).any())


@pytest.mark.parametrize("T", [40, 301])
def test_bad_expert_ids_in_the_tensor_memory_form(cuda, T):
    E, H, I, k = 4, 256, 128, 2
    p = ref.parts(E, H, I, 64, True, device=cuda)
    bank = bank_of(p)
    gen = torch.Generator().manual_seed(T)
    ids = torch.rand((T, E), generator=gen).argsort(1)[:, :k].int().contiguous().to(cuda)
    w = torch.rand((T, k), generator=gen).to(cuda)
    x = rows(T, H, 2, cuda)
    good = torch.ones_like(ids, dtype=torch.bool)
    good[0, 0] = good[7, 1] = good[T - 1, 0] = good[T - 1, 1] = False
    wrong = ids.clone()
    wrong[0, 0], wrong[7, 1], wrong[T - 1, 0], wrong[T - 1, 1] = 9, -1, 4, 2 ** 31 - 1
    y = ops.experts_w4(x, wrong, w, bank)
    with pytest.raises(ops.MoEKernelError, match="expert id"):
        ops.check_status(cuda)
    close(y, *ref.experts(p, x, ids, w * good))  # the good records are computed
    assert not bool(y[T - 1].any())
    ops.check_status(cuda)


@pytest.mark.parametrize("T", [3, 16, 40, 300])
def test_non_finite_rows_in_the_layer(cuda, T):
    """A token whose router logits are not numbers is routed somewhere; the others keep
    their rows, bit for bit, in every form of the layer."""
    E, H, I, k = 16, 256, 128, 4
    bank = bank_of(ref.parts(E, H, I, 128, True, seed=T, device=cuda))
    x = rows(T, H, 3, cuda)
    router = (torch.randn((E, H), generator=torch.Generator().manual_seed(T)) * 0.1).bfloat16().to(cuda)
    clean = ops.moe_layer_w4(x, router, bank, k)
    x[0, 3], x[T - 1, 9] = float("nan"), float("inf")
    y = ops.moe_layer_w4(x, router, bank, k)
    ops.check_status(cuda)
    assert torch.equal(y[1:T - 1], clean[1:T - 1])
    assert not bool(torch.isfinite(y[[0, T - 1]].float()).any())


# ------------------------------------------------------------------ what the forms round


FINE = 2.0 ** -12  # a weight, or a value of h, in fp16


def fine_down(m, v, h, e):
    """o = h Wd^T of expert e in 64 bits, and the bound of the tensor-memory form: fp32 sums,
    weights in fp16, activations of which fp16 holds all that is 2^-25 of the row's largest."""
    o = h.double() @ v[e].t()
    top = h.double().abs().amax(1, keepdim=True)
    return o, (ref.ACC * ref.operand_sums(m, h, e) + FINE * (h.double().abs() @ v[e].abs().t())
               + 2.0 ** -39 * top * v[e].abs().sum(1) + 2.0 ** -133)


def many(E, seed=0):
    """Offsets of at least TC_RECORDS rows per expert on average, ragged."""
    gen = torch.Generator().manual_seed(seed)
    c = torch.randint(0, 150, (E,), generator=gen)
    c[0], c[-1] = 129, 0
    return torch.cat([c.new_zeros(1), c.cumsum(0)])


@pytest.mark.parametrize("E,H,I,group,zeros", [(4, 256, 128, 64, True), (6, 2048, 768, 128, False),
                                               (3, 512, 192, 32, True), (2, 1024, 8192, 64, False)])
def test_many_records_do_not_round_the_weights_to_bf16(cuda, E, H, I, group, zeros):
    """Each product of many records is as near to 64 bits as its output's type lets it be."""
    p = ref.parts(E, H, I, group, zeros, seed=E, device=cuda)
    bank = bank_of(p)
    off = many(E).to(cuda)
    M = int(off[-1])
    assert M // E >= ref.TC_RECORDS
    x, hin = rows(M, H, 7, cuda), rows(M, I, 8, cuda)
    tiles, num, mt = ops.tiles_from_offsets(off, M)
    h = ops.grouped_w13_swiglu_w4(x, tiles, num, mt, bank)
    out = ops.grouped_w2_w4(hin, tiles, num, mt, bank)
    y = ops.sorted_experts_w4(x, off, bank)
    ops.check_status(cuda)
    vg, vu, vd = (ref.values(m) for m in p)
    for e in range(E):
        a, z = int(off[e]), int(off[e + 1])
        if a == z:
            continue
        g, u = x[a:z].double() @ vg[e].t(), x[a:z].double() @ vu[e].t()
        want = g * torch.sigmoid(g) * u
        rms_close(h[a:z], want, "h", False, f"h of expert {e}")
        o, do = fine_down(p[2], vd, hin[a:z], e)
        close(out[a:z], o, ref.BF16 * o.abs() + 1.01 * do, f"out of expert {e}")
        rms_close(out[a:z], o, "out", False, f"out of expert {e}")
        rms_close(y[a:z], want @ vd[e].t(), "out", False, f"rows of expert {e}")


@pytest.mark.parametrize("T,k", [(60, 2), (700, 3)])
def test_experts_of_many_records_round_twice(cuda, T, k):
    """The slot rows and the result, but neither the weights nor h, are rounded to bf16."""
    E, H, I = 4, 512, 256
    p = ref.parts(E, H, I, 64, True, seed=T, device=cuda)
    gen = torch.Generator().manual_seed(T)
    ids = torch.rand((T, E), generator=gen).argsort(1)[:, :k].int().contiguous().to(cuda)
    w = torch.rand((T, k), generator=gen).to(cuda)
    x = rows(T, H, 2, cuda)
    y = ops.experts_w4(x, ids, w, bank_of(p))
    ops.check_status(cuda)
    want, _ = ref.experts(p, x, ids, w)
    rel = ((y.double() - want).norm() / want.norm()).item()
    assert rel <= ref.BF16 * (2 / 3) ** 0.5 + 2.0 ** -12


@pytest.mark.parametrize("peak", [1e-30, 1e-3, 3e4, 1e30])
@pytest.mark.parametrize("group,zeros", [(64, False), (32, True)])
def test_activation_range_of_many_records(cuda, peak, group, zeros):
    """Rows of any magnitude that bf16 holds, rows of zeros, channels 2^20 times the others."""
    E, H, I = 2, 512, 128
    p = ref.parts(E, H, I, group, zeros, device=cuda)
    off = torch.tensor([0, 50, 120], device=cuda)
    h = rows(120, I, 8, cuda).float() * peak
    h[3] = 0.0
    h[6, 9] *= 2.0 ** 20 if peak < 1e10 else 1.0
    h[7, ::2] *= 2.0 ** -20 if peak > 1e-10 else 1.0
    h[60:70] *= 2.0 ** -60 if peak > 1e10 else 1.0
    h = h.bfloat16()
    tiles, num, mt = ops.tiles_from_offsets(off, 120)
    out = ops.grouped_w2_w4(h, tiles, num, mt, bank_of(p))
    ops.check_status(cuda)
    vd = ref.values(p[2])
    for e in range(E):
        a, z = int(off[e]), int(off[e + 1])
        o, do = fine_down(p[2], vd, h[a:z], e)
        close(out[a:z], o, ref.BF16 * o.abs() + 1.01 * do, f"expert {e}")


@pytest.mark.parametrize("T", [12, 120])
@pytest.mark.parametrize("group,zeros", [(128, False), (64, True), (32, False)])
def test_scales_of_any_size(cuda, T, group, zeros):
    """Experts, rows and groups whose scales are powers of two apart, rows of zeros, negative
    scales: every row keeps its own relative error in both forms of the products."""
    E, H, I = 2, 512, 256
    p = ref.parts(E, H, I, group, zeros, seed=group, device=cuda)
    gen = torch.Generator().manual_seed(T)
    for m in (0, 1, 2):
        codes, s, z = p[m]
        n = s.shape[1]
        by_row = torch.randint(-40, 8, (1, n, 1), generator=gen).double()
        by_row[:, ::3] = 0.0
        by_group = torch.randint(-6, 3, (E, n, s.shape[2]), generator=gen).double()
        by_expert = torch.tensor([0.0, -30.0 if m else 20.0]).view(E, 1, 1).double()
        f = torch.exp2(by_row + by_group + by_expert).to(cuda)
        f[:, 5] = 0.0
        f[:, 7] *= -1.0
        s.copy_((s.double() * f).bfloat16())
    bank = bank_of(p)
    off = torch.tensor([0, T // 2, T], device=cuda)
    x, hin = rows(T, H, 7, cuda), rows(T, I, 8, cuda)
    tiles, num, mt = ops.tiles_from_offsets(off, T)
    h = ops.grouped_w13_swiglu_w4(x, tiles, num, mt, bank)
    out = ops.grouped_w2_w4(hin, tiles, num, mt, bank)
    y = ops.sorted_experts_w4(x, off, bank)
    ops.check_status(cuda)
    vg, vu, vd = (ref.values(m) for m in p)
    for e in range(E):
        a, z = int(off[e]), int(off[e + 1])
        want, bound = ref.swiglu_rows(p[0], p[1], vg, vu, x[a:z], e, False)
        g, u = x[a:z].double() @ vg[e].t(), x[a:z].double() @ vu[e].t()
        fg, fu = (FINE * (x[a:z].double().abs() @ v[e].abs().t()) for v in (vg, vu))
        wide = bound + 1.1 * fg * (u.abs() + fu) + (g * torch.sigmoid(g)).abs() * fu + 2.0 ** -133
        close(h[a:z], want, wide * 1.01, f"h of expert {e}")
        o, do = fine_down(p[2], vd, hin[a:z], e)
        close(out[a:z], o, ref.BF16 * o.abs() + 1.01 * do, f"out of expert {e}")
        # h in bf16 (few rows) or fp16 of the row's largest value (many), then the down product
        dh = wide * 1.01 + 2.0 ** -39 * want.abs().amax(1, keepdim=True)
        ws, ds = fine_down(p[2], vd, want, e)
        close(y[a:z], ws, ref.BF16 * ws.abs() + 1.02 * (ds + dh @ vd[e].abs().t()), f"y of expert {e}")


@pytest.mark.parametrize("x_exp,s_exp", [(-112, 20), (-100, -8), (-108, -28), (-60, -60), (0, -90),
                                         (0, 40), (90, 12), (118, -30), (60, 30)])
def test_far_ranges_of_many_records(cuda, x_exp, s_exp):
    """Activations and scales that lie far out on either side, together with rows of zeros on
    both: results that bf16 holds are right, and zeros stay zeros."""
    E, H, I = 2, 256, 128
    p = ref.parts(E, H, I, 64, True, device=cuda)
    codes, scales, zeros = p[2]
    scales.copy_((scales.double() * 2.0 ** s_exp).bfloat16())
    codes[:, 3] = zeros[:, 3].repeat_interleave(64, -1)  # weights of zero under large scales
    scales[:, 9] = 0.0
    bank = bank_of(p)
    off = torch.tensor([0, 30, 70], device=cuda)
    h = rows(70, I, 8, cuda).double() * 2.0 ** x_exp
    h[2] = 0.0
    h[33, 1:] = 0.0
    h = h.bfloat16()
    tiles, num, mt = ops.tiles_from_offsets(off, 70)
    out = ops.grouped_w2_w4(h, tiles, num, mt, bank)
    ops.check_status(cuda)
    assert not bool(out[2].any()) and not bool(out[:, 3].any()) and not bool(out[:, 9].any())
    vd = ref.values(p[2])
    for e in range(E):
        a, z = int(off[e]), int(off[e + 1])
        o, do = fine_down(p[2], vd, h[a:z], e)
        assert bool((o.abs() < 3e38).all())
        close(out[a:z], o, ref.BF16 * o.abs() + 1.01 * do, f"expert {e}")


def test_many_records_on_a_bank_without_fine_scales(cuda):
    """A bank of codes and scales alone, as a caller of the C ABI may pack it: products of
    many records stream, with the weights exact."""
    E, H, I = 4, 256, 192
    p = ref.parts(E, H, I, 64, True, device=cuda)
    full = bank_of(p)
    plain = W4Experts(full.w13[:2], full.w2[:2], E, H, I, 64, True)
    off = many(E).to(cuda)
    M = int(off[-1])
    x = rows(M, H, 3, cuda)
    y, z = (ops.sorted_experts_w4(x, off, b) for b in (plain, full))
    ops.check_status(cuda)
    owner = torch.repeat_interleave(torch.arange(E, device=cuda), off.diff())
    want, bound = ref.experts(p, x, owner[:, None], torch.ones((M, 1), device=cuda))
    close(y, want, bound)
    close(z, want, bound)
    rms_close(y, z.double(), "y", False)
    tiles, num, mt = ops.tiles_from_offsets(off, M)
    h = ops.grouped_w13_swiglu_w4(x, tiles, num, mt, plain)
    rms_close(h, ops.grouped_w13_swiglu_w4(x, tiles, num, mt, full).double(), "y", False)
    ops.check_status(cuda)
    # the C calls without a workspace stream too, on any bank
    q, lib = ops._p, ops._native.load()
    again = torch.empty_like(h)
    assert lib.moe_grouped_w13_swiglu_w4(q(x), M, None, 1, M, q(tiles), q(num), mt, full.native,
                                         q(again), q(ops.status_word(cuda)), ops._stream(cuda)) == 0
    assert torch.equal(again, h)
    out = ops.grouped_w2_w4(h, tiles, num, mt, plain)
    again = torch.empty_like(out)
    assert lib.moe_grouped_w2_w4(q(h), M, q(tiles), q(num), mt, full.native, None, None, q(again),
                                 M, q(ops.status_word(cuda)), ops._stream(cuda)) == 0
    assert torch.equal(again, out)
    ops.check_status(cuda)


@pytest.mark.parametrize("T", [23, 24, 31, 32, 33])
def test_shard_beside_the_choice_of_form(cuda, T):
    """Many records for each expert that the bank holds, but few for each of all experts, and
    the first batches on the other side: the workspace serves both."""
    E, H, I, k = 4, 256, 128, 4
    p = ref.parts(E, H, I, 64, True, seed=T, device=cuda)
    bank = bank_of(p)
    gen = torch.Generator().manual_seed(T)
    ids = torch.rand((T, 16), generator=gen).argsort(1)[:, :k].int().contiguous().to(cuda)
    w = torch.randn((T, k), generator=gen).to(cuda)
    x = rows(T, H, 2, cuda)
    ws = torch.empty(ops.experts_w4_workspace_bytes(T, k, bank), dtype=torch.uint8, device=cuda)
    y = ops.experts_w4(x, ids, w, bank, num_experts=16, e_begin=6, workspace=ws)
    ops.check_status(cuda)
    close(y, *ref.experts(p, x, ids, w, e_begin=6, num_experts=16))


def test_bank_into_another(cuda):
    """The memory of a bank of the same sizes and form is taken over; of any other it is not."""
    p, q = (ref.parts(2, 128, 64, 32, True, seed=s, device=cuda) for s in (0, 1))
    first, want = bank_of(p), bank_of(q)
    plain = W4Experts(first.w13[:2], first.w2[:2], 2, 128, 64, 32, True)
    other = bank_of(ref.parts(2, 128, 64, 32, False, device=cuda))
    for into, takes in ((plain, False), (other, False), (first, True)):
        was = [t.data_ptr() for t in (*into.w13, *into.w2)]
        got = W4Experts.from_codes(*q, into=into)
        assert ([t.data_ptr() for t in (*got.w13, *got.w2)] == was) == takes
        assert all(torch.equal(a, b) for a, b in zip((*got.w13, *got.w2), (*want.w13, *want.w2)))


def test_first_call_under_a_capture(cuda):
    """The status word does not become the graph's: it is zero before any replay, and a replay
    does not clear what was reported."""
    here = os.path.dirname(os.path.abspath(__file__))
    run = subprocess.run([sys.executable, os.path.join(here, "first_in_capture.py")],
                         capture_output=True, text=True, timeout=120)
    assert run.returncode == 0 and run.stdout.split()[-1:] == ["ok"], run.stdout + run.stderr
