"""The 4-bit experts and the block norm where a model calls them: the modules, runs of
the operators together, and shapes at the edges of the kernels' forms."""

import os
import sys

import pytest
import torch

import w4_reference as ref
from moe_inference_verify_microbench_b200 import (PermutedSparseMoE, W4Experts, dequantize_w4,
                                                  fused_moe_forward_w4, ops, quantize_w4)
from test_gpu_ep import _init, _need, _spawn
from test_gpu_w4 import bank_of, close, rms_close, rows

HERE = os.path.dirname(os.path.abspath(__file__))
pytestmark = pytest.mark.gpu


def module(cuda, H=256, I=128, E=16, k=4, **options):
    torch.manual_seed(5)
    mod = PermutedSparseMoE(H, I, E, k, expert_weights="w4", **options)
    return mod.to(device=cuda, dtype=torch.bfloat16)


@pytest.mark.parametrize("group,symmetric", [(32, False), (64, True), (128, False)])
def test_quantize_and_pack(cuda, group, symmetric):
    """Codes taken on the GPU and packed expert by expert are those of the CPU."""
    E, H, I = 3, 256, 384
    gen = torch.Generator().manual_seed(group)
    w = [(torch.randn(s, generator=gen) * 0.1).bfloat16() for s in ((E, I, H), (E, I, H), (E, H, I))]
    here = W4Experts.quantize(*(t.to(cuda) for t in w), group, symmetric)
    parts = [quantize_w4(t, group, symmetric) for t in w]
    there = bank_of([tuple(None if t is None else t.to(cuda) for t in p) for p in parts])
    assert here.has_zeros == there.has_zeros == (not symmetric)
    for a, b in zip((*here.w13, *here.w2), (*there.w13, *there.w2)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("symmetric", [True, False])
@pytest.mark.parametrize("shape", [(1,), (2, 3), (2, 20), (300,)])
def test_module(cuda, symmetric, shape):
    H, E, k = 256, 16, 4
    mod = module(cuda, H=H, group_size=64, symmetric=symmetric)
    x = rows(torch.Size(shape).numel(), H, 3, cuda)
    with torch.no_grad():
        y = mod(x.reshape(*shape, H))
    ids, w, _ = ops.router_topk(x, mod.gate.weight, k)
    ops.check_status(cuda)
    parts = [quantize_w4(t, 64, symmetric) for t in mod.pack()]
    want, bound = ref.experts(parts, x, ids, w)
    assert y.shape == (*shape, H)
    close(y.reshape(-1, H), want, bound)
    rms_close(y.reshape(-1, H), want, "y", x.shape[0] * k // E >= ref.TC_RECORDS)


def test_module_follows_its_weights(cuda):
    mod = module(cuda, group_size=64)
    x = rows(5, 256, 3, cuda)
    with torch.no_grad():
        y = mod(x)
        bank = mod.experts_4bit()
        assert mod.experts_4bit() is bank
        mod.pack()[2].mul_(2.0)                    # through the stacked tensor: noticed
        assert mod.experts_4bit() is not bank
        assert torch.equal(mod(x).float(), 2.0 * y.float())  # scales of twice the size
        mod.experts[3].down_proj.weight.zero_()    # through one expert: on request
        bank = mod.experts_4bit(refresh=True)
        assert not bool(bank.w2[1].view(16, -1)[3].any())
        mod.to(cuda)
        assert mod.experts_4bit() is not bank
    assert mod(torch.empty(2, 0, 256, dtype=torch.bfloat16, device=cuda)).shape == (2, 0, 256)
    ops.check_status(cuda)


@pytest.mark.parametrize("T", [1, 7, 40, 300])
def test_run_of_the_operators(cuda, T):
    """norm -> router and 4-bit experts -> norm, as a decoder layer's second half, each
    step against 64 bits on the step's own inputs, and replayed from a graph."""
    E, H, I, k = 16, 512, 256, 4
    p = ref.parts(E, H, I, 128, False, device=cuda)
    bank = bank_of(p)
    gen = torch.Generator().manual_seed(T)
    vec = lambda: (torch.rand(H, generator=gen) + 0.5).to(cuda)
    router = (torch.randn((E, H), generator=gen) * 0.08).bfloat16().to(cuda)
    x, a = rows(T, H, 1, cuda), rows(T, H, 2, cuda)
    w1, w2, w3, w4, gate = vec(), vec(), vec(), vec(), vec()

    def run():
        h, n = ops.block_norm(x, a, w1, w2, 1e-6, gate=gate, gate_act="sigmoid")
        m = ops.moe_layer_w4(n, router, bank, k)
        return h, n, m, *ops.block_norm(h, m, w3, w4, 1e-6, residual_scale=0.5)

    h, n, m, y, z = run()
    ids, w, _ = ops.router_topk(n, router, k)
    ops.check_status(cuda)
    wh, wn, dh, dn = ref.block_norm(x, a, w1, w2, 1e-6, gate, "sigmoid", 1.0)
    close(h, wh, dh)
    close(n, wn, dn)
    close(m, *ref.experts(p, n, ids, w))
    wy, wz, dy, dz = ref.block_norm(h, m, w3, w4, 1e-6, None, "none", 0.5)
    close(y, wy, dy)
    close(z, wz, dz)
    side = torch.cuda.Stream(cuda)
    side.wait_stream(torch.cuda.current_stream(cuda))
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream(cuda).wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    for _ in range(2):
        for t in out:
            t.zero_()
        graph.replay()
        for t, was in zip(out, (h, n, m, y, z)):
            assert torch.equal(t, was)
    x.copy_(rows(T, H, 9, cuda))  # other inputs in the same places
    graph.replay()
    for t, was in zip(out, run()):
        assert torch.equal(t, was)


@pytest.mark.parametrize("counts", [[0, 3, 1, 9], [128, 0, 60, 129]])
@pytest.mark.parametrize("extra", [0, 1, 300])
def test_rows_past_the_last_expert(cuda, counts, extra):
    """Zero in the output of the sorted call, in both forms of the product."""
    E, H, I = 4, 256, 192
    p = ref.parts(E, H, I, 64, True, device=cuda)
    off = torch.tensor([0] + counts).cumsum(0).to(cuda)
    M = int(off[-1])
    x = rows(M + extra, H, 3, cuda)
    out = torch.full((M + extra, H), 7.0, dtype=torch.bfloat16, device=cuda)
    y = ops.sorted_experts_w4(x, off, bank_of(p), out=out)
    ops.check_status(cuda)
    assert y.data_ptr() == out.data_ptr() and not bool(y[M:].any())
    owner = torch.repeat_interleave(torch.arange(E, device=cuda), off.diff())
    # the form goes by all rows of the call
    fake = torch.full((M + extra, 1), -1, device=cuda)
    fake[:M, 0] = owner
    want, bound = ref.experts(p, x, fake, torch.ones((M + extra, 1), device=cuda))
    close(y, want, bound)
    assert torch.equal(y, fused_moe_forward_w4(x, off, bank_of(p)))


@pytest.mark.parametrize("E,H,I,k,T", [(16, 256, 128, 4, 16), (32, 4096, 128, 2, 2), (16, 256, 64, 1, 1),
                                       (48, 512, 384, 8, 8), (16, 2560, 64, 4, 13)])
def test_layer_edges(cuda, E, H, I, k, T):
    """The one-kernel layer at its most tokens and records and with several row tiles
    for a CTA; the same tokens alone and in a batch give the same rows."""
    p = ref.parts(E, H, I, 64, False, seed=T, device=cuda)
    bank = bank_of(p)
    x = rows(T, H, 3, cuda)
    router = (torch.randn((E, H), generator=torch.Generator().manual_seed(T)) * 1.8
              * H ** -0.5).bfloat16().to(cuda)
    y = ops.moe_layer_w4(x, router, bank, k)
    ids, w, _ = ops.router_topk(x, router, k)
    ops.check_status(cuda)
    want, bound = ref.experts(p, x, ids, w)
    close(y, want, bound)
    rms_close(y, want, "y", False)


@pytest.mark.parametrize("T", [9, 12, 16])
def test_layer_past_the_one_kernel_form(cuda, T):
    """More than 64 records of at most 16 tokens: the rows are those of a larger batch
    (the records of a token are summed in the same order in any of them)."""
    E, H, I, k = 64, 512, 128, 8
    p = ref.parts(E, H, I, 128, True, seed=T, device=cuda)
    bank = bank_of(p)
    x = rows(24, H, 3, cuda)
    router = (torch.randn((E, H), generator=torch.Generator().manual_seed(T)) * 0.08).bfloat16().to(cuda)
    y = ops.moe_layer_w4(x[:T].contiguous(), router, bank, k)
    more = ops.moe_layer_w4(x, router, bank, k)
    ids, w, _ = ops.router_topk(x, router, k)
    ops.check_status(cuda)
    want, bound = ref.experts(p, x, ids, w)
    close(more, want, bound)
    assert torch.equal(y, more[:T])


@pytest.mark.parametrize("H,I,group,zeros", [(64, 512, 64, False), (192, 320, 32, True), (320, 64, 64, True)])
def test_many_units(cuda, H, I, group, zeros):
    """More units than CTAs at odd numbers of 64-column blocks, entries of 1 to 128 rows
    in turn on one CTA, row blocks that end inside a unit."""
    E = 160
    p = ref.parts(E, H, I, group, zeros, device=cuda)
    bank = bank_of(p)
    gen = torch.Generator().manual_seed(H)
    counts = torch.randint(0, 129, (E,), generator=gen)
    counts[::7] = 0
    counts[5::11] = 1
    off = torch.cat([counts.new_zeros(1), counts.cumsum(0)]).to(cuda)
    M = int(off[-1])
    assert M // E >= ref.TC_RECORDS
    x = rows(M, H, 7, cuda)
    y = ops.sorted_experts_w4(x, off, bank)
    again = ops.sorted_experts_w4(x, off, bank)
    ops.check_status(cuda)
    owner = torch.repeat_interleave(torch.arange(E, device=cuda), off.diff())
    want, bound = ref.experts(p, x, owner[:, None], torch.ones((M, 1), device=cuda))
    close(y, want, bound)
    assert torch.equal(y, again)


def test_entries_of_more_than_128_rows_are_reported(cuda):
    E, H, I = 2, 64, 64
    bank = bank_of(ref.parts(E, H, I, 64, False, device=cuda))
    M = 200
    tiles = torch.tensor([[0, 0, 200, 0]], dtype=torch.int32, device=cuda)
    num = torch.ones(1, dtype=torch.int32, device=cuda)
    out = torch.full((M, I), 7.0, dtype=torch.bfloat16, device=cuda)
    ops.grouped_w13_swiglu_w4(rows(M, H, 1, cuda), tiles, num, 1, bank, out=out)
    with pytest.raises(ops.MoEKernelError):
        ops.check_status(cuda)
    assert bool((out == 7.0).all())


def _block_worker(rank, world, port, q):
    sys.path.insert(0, HERE)
    sys.path.insert(0, os.path.dirname(HERE))
    import torch.distributed as dist
    from moe_inference_verify_microbench_b200.hybrid import HybridBlock

    dev = _init(rank, world, port)
    try:
        H, I, E, k, nh, nkv, hd, scale = 512, 256, 16, 4, 8, 2, 64, 0.5
        g = torch.Generator(device=dev)
        g.manual_seed(21)
        r = lambda *s, sc=0.04: (torch.randn(*s, generator=g, device=dev) * sc).to(torch.bfloat16)
        blocks = []
        for act in ("sigmoid", None):
            with torch.device(dev):
                blk = HybridBlock(H, I, nh, nkv, hd, E, k, world, rank, None, world, rank, None,
                                  post_norm=True, gate_act=act, residual_scale=scale)
            blk = blk.to(torch.bfloat16)
            gates = {} if act is None else {"attn_gate": r(H, sc=1.0), "moe_gate": r(H, sc=1.0)}
            blk.weight_loader(1.0 + r(H, sc=0.1), r(nh * hd, H), r(nkv * hd, H), r(nkv * hd, H),
                              r(H, nh * hd), 1.0 + r(H, sc=0.1), r(E, H), list(r(E, I, H)),
                              list(r(E, I, H)), list(r(E, H, I)),
                              attn_post_norm_weight=1.0 + r(H, sc=0.1),
                              moe_post_norm_weight=1.0 + r(H, sc=0.1), **gates)
            blocks.append(blk)
        first, second = blocks
        x = r(2, 24, H, sc=1.0)
        with torch.no_grad():
            y = first(x)
            y2, n = first(x, next_norm=second.attn_norm)
            end, chained = second(y), second(y2, normed=n)
            # the same with the harness norms
            def plain(blk, x):
                one = lambda v: 1.0 if v is None else torch.sigmoid(v.float())
                ga, gm = (getattr(blk, a, None) for a in ("attn_gate", "moe_gate"))
                a = blk.attn_post_norm(blk.attn(blk.attn_norm(x))).float()
                h = (x.float() + scale * one(ga) * a).to(x.dtype)
                m = blk.moe_post_norm(blk.moe(blk.moe_norm(h))).float()
                return (h.float() + scale * one(gm) * m).to(x.dtype)
            want, wend = plain(first, x), plain(second, y)
        torch.cuda.synchronize()
        ops.check_status(dev)

        def frac(got, want):
            err = ((got.float() - want.float()).abs().amax(-1) / want.float().abs().amax(-1))
            return float((err <= 2e-2).float().mean())
        q.put((rank, [frac(y, want), frac(end, wend), frac(chained, end),
                      float(torch.equal(y, y2))]))
        dist.barrier()
    finally:
        dist.destroy_process_group()


def test_block_with_norms_after_its_branches(cuda):
    """HybridBlock(post_norm=True) on ``ops.block_norm`` against the harness norms, alone and
    chained (tp = ep = 1, one process)."""
    _need(1)
    for rank, fracs in _spawn(_block_worker, 1, (29975,)):
        # a norm's last bit may flip a top-k boundary
        assert min(fracs[:3]) >= 0.9 and fracs[3] == 1.0, (rank, fracs)


def test_dequantised_weights(cuda):
    """The values that stand behind a bank, from the helper that a loader would use."""
    p = ref.parts(2, 128, 64, 32, True, device=cuda)
    for m in p:
        assert torch.equal(dequantize_w4(*m).double(), ref.values(m))
