"""The 4-bit expert operators and the block norm against plain 64-bit forms."""

from __future__ import annotations

import pytest
import torch

import w4_reference as ref
from moe_inference_verify_microbench_b200 import W4Experts, fused_moe_forward_w4, ops

pytestmark = pytest.mark.gpu


def close(got, want, bound, what=""):
    err = (got.double() - want).abs()
    worst = (err / bound).max().item() if err.numel() else 0.0
    assert torch.isfinite(got.float()).all(), f"{what}: not finite"
    assert worst <= 1.0, f"{what}: an element is {worst:.3g} times its bound off"


def rms_close(got, want, parts, rounded, what=""):
    """Each rounding to bf16 is BF16 / sqrt(3) of its value in the mean at most, and they
    are independent; 2^-12 for the fp32 sums (random signs leave far less of their bound)."""
    rel = ((got.double() - want).norm() / want.norm()).item()
    most = ref.BF16 * (ref.roundings(parts, rounded) / 3) ** 0.5 + 2.0 ** -12
    assert rel <= most, f"{what}: relative error {rel:.3g}, at most {most:.3g} expected"


def bank_of(p):
    return W4Experts.from_codes(*p)


def rows(T, H, seed, device):
    return torch.randn((T, H), generator=torch.Generator().manual_seed(seed)).bfloat16().to(device)


def unpack(packed, E, N, K, pair):
    """Codes [E, N, K] of each packed matrix, from the documented layout."""
    r = 8 if pair else 16
    q = packed.view(E, N // r, K // 64, 8, 4, 4, 4)  # tile, block, g, t, word, byte
    nib = torch.stack([q & 15, q >> 4], -1).reshape(*q.shape[:-1], 8)  # nibble order
    cols = nib.reshape(*nib.shape[:-1], 2, 4)  # [.., low or high column of the pair, i]
    out = []
    for half in (0, 1):  # row g, row g + 8: words 2 half, 2 half + 1
        w = cols[..., 2 * half:2 * half + 2, :, :]  # E, tile, block, g, t, word, low/high, i
        w = w.permute(0, 1, 3, 2, 5, 7, 4, 6)       # E, tile, g, block, word, i, t, low/high
        out.append(w.reshape(E, N // r, 8, K))
    if pair:
        return [o.reshape(E, N, K) for o in out]
    return [torch.stack(out, 2).reshape(E, N, K)]


@pytest.mark.parametrize("E,H,I,group,zeros", [(2, 64, 64, 64, False), (3, 256, 192, 32, True),
                                               (1, 512, 128, 128, True)])
def test_packed_layout(cuda, E, H, I, group, zeros):
    p = ref.parts(E, H, I, group, zeros, device=cuda)
    b = bank_of(p)
    g, u = unpack(b.w13[0], E, I, H, True)
    assert torch.equal(g, p[0][0]) and torch.equal(u, p[1][0])
    assert torch.equal(unpack(b.w2[0], E, H, I, False)[0], p[2][0])
    n = 4 if zeros else 2
    s13 = b.w13[1].view(E, I // 8, H // group, 8, n)
    s2 = b.w2[1].view(E, H // 16, I // group, 8, n)
    assert torch.equal(s13[..., 0].permute(0, 1, 3, 2).reshape(E, I, -1), p[0][1])
    assert torch.equal(s13[..., 1].permute(0, 1, 3, 2).reshape(E, I, -1), p[1][1])
    assert torch.equal(s2[..., :2].permute(0, 1, 4, 3, 2).reshape(E, H, -1), p[2][1])
    if zeros:  # kept as 128 + z
        z13, z2 = (t.float() - 128 for t in (s13[..., 3], s2[..., 2:]))
        assert torch.equal(z13.permute(0, 1, 3, 2).reshape(E, I, -1), p[1][2].float())
        assert torch.equal(z2.permute(0, 1, 4, 3, 2).reshape(E, H, -1), p[2][2].float())


def test_codes_above_15_are_refused(cuda):
    p = ref.parts(1, 64, 64, 64, True, device=cuda)
    p[1][0][0, 5, 7] = 16
    with pytest.raises(ValueError, match="0..15"):
        bank_of(p)
    p = ref.parts(1, 64, 64, 64, True, device=cuda)
    p[2][2][0, 63, 0] = 255
    with pytest.raises(ValueError, match="0..15"):
        bank_of(p)


# hidden and intermediate sizes that cut differently over the warps (K / 64 blocks of
# 1, 2, 3, 6, 12, 20, 32, 40 and 128), every group, with and without zero points
SHAPES = [(4, 64, 64, 64, False), (3, 128, 64, 32, True), (5, 192, 384, 64, True),
          (4, 768, 1280, 128, False), (6, 2048, 768, 128, False), (3, 2560, 192, 32, False),
          (2, 2048, 192, 64, True), (1, 8192, 128, 128, False), (1, 8192, 64, 32, True),
          (2, 1024, 8192, 64, False)]
# ragged: empty experts, one row, around the 8, 16, 32 and 128 row steps
COUNTS = [0, 1, 7, 8, 9, 16, 17, 33, 0, 2, 129, 40]
MANY = [128, 0, 60, 64, 65, 1, 257, 17, 96, 80]  # at least TC_RECORDS in the mean


def offsets_of(E, device, shift=0):
    steps = COUNTS if shift < 100 else MANY
    c = [steps[(e + shift) % len(steps)] for e in range(E)]
    off = torch.tensor([0] + c).cumsum(0)
    return off.to(device), int(off[-1])


@pytest.mark.parametrize("E,H,I,group,zeros", SHAPES)
@pytest.mark.parametrize("shift", [1, 6, 10, 100, 104, 106])
def test_grouped_products(cuda, E, H, I, group, zeros, shift):
    """Both grouped products, each from exact inputs."""
    p = ref.parts(E, H, I, group, zeros, seed=shift, device=cuda)
    bank = bank_of(p)
    off, M = offsets_of(E, cuda, shift)
    x = rows(M, H, 7, cuda)
    tiles, num, mt = ops.tiles_from_offsets(off, M)
    h = ops.grouped_w13_swiglu_w4(x, tiles, num, mt, bank)
    hin = rows(M, I, 8, cuda)
    scale = torch.rand(M, generator=torch.Generator().manual_seed(3)).to(cuda) + 0.5
    perm = torch.randperm(M, generator=torch.Generator().manual_seed(4)).int().to(cuda)
    out = torch.full((M + 2, H), 7.0, dtype=torch.bfloat16, device=cuda)
    sc = torch.cat([scale, scale.new_zeros(2)])
    ops.grouped_w2_w4(hin, tiles, num, mt, bank, row_map=perm, slot_scale=sc, out=out)
    ops.check_status(cuda)
    vg, vu, vd = (ref.values(m) for m in p)
    rounded = M // E >= ref.TC_RECORDS
    for e in range(E):
        a, z = int(off[e]), int(off[e + 1])
        if a == z:
            continue
        want, bound = ref.swiglu_rows(p[0], p[1], vg, vu, x[a:z], e, rounded)
        close(h[a:z], want, bound, f"h of expert {e}")
        rms_close(h[a:z], want, "h", rounded, f"h of expert {e}")
        o, do = ref.down_rows(p[2], vd, hin[a:z], e, rounded)
        m = perm[a:z].long()
        s = scale[m].double().unsqueeze(1)
        close(out[m], s * o, ref.BF16 * (s * o).abs() + 1.01 * s * do + 1e-30, f"out of expert {e}")
        rms_close(out[m], s * o, "out", rounded, f"out of expert {e}")
    assert bool((out[M:] == 7.0).all()), "rows that no record maps to are left as they were"


@pytest.mark.parametrize("peak", [1e-30, 1e-3, 3e4, 1e30])
@pytest.mark.parametrize("group,zeros", [(64, False), (32, True)])
def test_activation_range(cuda, peak, group, zeros):
    """Rows of any magnitude that bf16 holds, beside rows of zeros, with channels 2^20
    times the others."""
    E, H, I = 2, 512, 128
    p = ref.parts(E, H, I, group, zeros, device=cuda)
    bank = bank_of(p)
    off = torch.tensor([0, 5, 12], device=cuda)
    h = rows(12, I, 8, cuda).float() * peak
    h[3] = 0.0
    h[6, 9] *= 2.0 ** 20 if peak < 1e10 else 1.0
    h[7, ::2] *= 2.0 ** -20 if peak > 1e-10 else 1.0
    h = h.bfloat16()
    tiles, num, mt = ops.tiles_from_offsets(off, 12)
    out = ops.grouped_w2_w4(h, tiles, num, mt, bank)
    ops.check_status(cuda)
    vd = ref.values(p[2])
    for e in range(E):
        a, z = int(off[e]), int(off[e + 1])
        o, do = ref.down_rows(p[2], vd, h[a:z], e, False)
        close(out[a:z], o, ref.BF16 * o.abs() + 1.01 * do + 2.0 ** -133, f"expert {e}")
        rms_close(out[a:z], o, "out", False, f"expert {e}")


@pytest.mark.parametrize("index_div", [1, 3])
def test_grouped_gather(cuda, index_div):
    E, H, I = 4, 256, 128
    p = ref.parts(E, H, I, 64, False, device=cuda)
    bank = bank_of(p)
    off, M = offsets_of(E, cuda, 4)
    src = rows(11, H, 5, cuda)
    index = torch.randint(0, 11 * index_div, (M,), generator=torch.Generator().manual_seed(1)).int().to(cuda)
    tiles, num, mt = ops.tiles_from_offsets(off, M)
    h = ops.grouped_w13_swiglu_w4(src, tiles, num, mt, bank, index=index, index_div=index_div)
    same = ops.grouped_w13_swiglu_w4(src[(index // index_div).long()].contiguous(), tiles, num, mt, bank)
    ops.check_status(cuda)
    assert torch.equal(h, same)


@pytest.mark.parametrize("E,H,I,group,zeros,k,T", [
    (16, 256, 128, 64, False, 4, 1), (16, 256, 128, 32, True, 8, 3), (16, 512, 192, 64, True, 2, 40),
    (8, 2048, 768, 128, False, 8, 17), (16, 1024, 384, 128, False, 8, 300),
    (4, 256, 128, 64, False, 3, 700), (128, 256, 128, 64, False, 8, 33)])
def test_experts(cuda, E, H, I, group, zeros, k, T):
    p = ref.parts(E, H, I, group, zeros, seed=T, device=cuda)
    bank = bank_of(p)
    gen = torch.Generator().manual_seed(T)
    ids = torch.rand((T, E), generator=gen).argsort(1)[:, :k].int().contiguous().to(cuda)
    w = torch.rand((T, k), generator=gen).to(cuda)
    x = rows(T, H, 2, cuda)
    y = ops.experts_w4(x, ids, w, bank)
    ops.check_status(cuda)
    want, bound = ref.experts(p, x, ids, w)
    close(y, want, bound)
    rms_close(y, want, "y", T * k // E >= ref.TC_RECORDS)
    assert torch.equal(y, ops.experts_w4(x, ids, w, bank)), "the same call twice"


def test_experts_shard_and_repeated_ids(cuda):
    """A bank of experts 6..9 of 16: other records add nothing, a token without any
    gets zeros, and one expert may be picked twice by a token."""
    E, H, I, k, T = 4, 256, 128, 4, 50
    p = ref.parts(E, H, I, 64, True, device=cuda)
    bank = bank_of(p)
    gen = torch.Generator().manual_seed(9)
    ids = torch.randint(0, 16, (T, k), generator=gen).int()
    ids[3] = torch.tensor([0, 1, 2, 15])   # none of the bank's
    ids[4] = torch.tensor([7, 7, 7, 7])
    ids = ids.to(cuda)
    w = torch.randn((T, k), generator=gen).to(cuda)
    x = rows(T, H, 2, cuda)
    out = torch.full((T, H), float("nan"), dtype=torch.bfloat16, device=cuda)
    y = ops.experts_w4(x, ids, w, bank, num_experts=16, e_begin=6, out=out)
    ops.check_status(cuda)
    assert y.data_ptr() == out.data_ptr()
    assert not bool(y[3].any())
    want, bound = ref.experts(p, x, ids, w, e_begin=6, num_experts=16)
    close(y, want, bound)


@pytest.mark.parametrize("E,H,I,group,zeros,k,T,bias,norm", [
    (16, 256, 128, 64, False, 4, 1, False, True), (16, 256, 128, 64, True, 4, 5, True, False),
    (128, 2048, 768, 128, False, 8, 1, False, True), (32, 2048, 192, 32, True, 8, 7, True, True),
    (32, 1024, 256, 64, False, 1, 64, False, True), (64, 512, 128, 64, False, 6, 33, False, False),
    (16, 256, 128, 64, False, 2, 500, True, True), (16, 8192, 64, 64, False, 2, 3, False, True)])
def test_layer(cuda, E, H, I, group, zeros, k, T, bias, norm):
    p = ref.parts(E, H, I, group, zeros, seed=T, device=cuda)
    bank = bank_of(p)
    gen = torch.Generator().manual_seed(T)
    x = rows(T, H, 3, cuda)
    router = (torch.randn((E, H), generator=gen) * 1.8 * H ** -0.5).bfloat16().to(cuda)
    b = torch.randn(E, generator=gen).to(cuda) if bias else None
    y = ops.moe_layer_w4(x, router, bank, k, norm_topk_prob=norm, bias=b)
    ids, w, _ = ops.router_topk(x, router, k, norm, b)
    ops.check_status(cuda)
    want, bound = ref.experts(p, x, ids, w)  # under the framework's own routing
    close(y, want, bound)
    rms_close(y, want, "y", T * k // E >= ref.TC_RECORDS)
    rid, rw = ref.route(x, router, b, k, norm)
    same = (rid == ids).all(1)  # the rest: logits within rounding of a tie
    assert same.double().mean() >= 0.98
    # a logit may round to the neighbouring bf16 value where its fp32 sum is at a border;
    # a weight below 2^-126 is not held by the fp32 output (e^-160 occurs: 1.6e-70 reads 0)
    assert ((rw - w.double()).abs()[same] <= 2.0 ** -5 * rw[same] + 2.0 ** -126).all()


def test_layer_large_batch_equals_experts(cuda):
    E, H, I, k, T = 16, 512, 256, 4, 1500
    p = ref.parts(E, H, I, 128, False, device=cuda)
    bank = bank_of(p)
    x = rows(T, H, 3, cuda)
    router = (torch.randn((E, H), generator=torch.Generator().manual_seed(1)) * 0.08).bfloat16().to(cuda)
    y = ops.moe_layer_w4(x, router, bank, k)
    ids, w, _ = ops.router_topk(x, router, k)
    z = ops.experts_w4(x, ids, w, bank)
    ops.check_status(cuda)
    assert torch.equal(y, z)


def test_fused_moe_forward_w4(cuda):
    E, H, I = 12, 256, 192
    p = ref.parts(E, H, I, 64, True, device=cuda)
    bank = bank_of(p)
    off, M = offsets_of(E, cuda)
    x = rows(M + 5, H, 3, cuda)  # five rows past the last expert
    y = fused_moe_forward_w4(x, off, bank)
    ops.check_status(cuda)
    owner = torch.repeat_interleave(torch.arange(E, device=cuda), off.diff())
    want, bound = ref.experts(p, x[:M], owner[:, None], torch.ones((M, 1), device=cuda))
    close(y[:M], want, bound)
    assert not bool(y[M:].any())


def test_empty_batches(cuda):
    p = ref.parts(16, 256, 128, 64, False, device=cuda)
    bank = bank_of(p)
    x = torch.empty((0, 256), dtype=torch.bfloat16, device=cuda)
    ids = torch.empty((0, 4), dtype=torch.int32, device=cuda)
    assert ops.experts_w4(x, ids, ids.float(), bank).shape == (0, 256)
    router = torch.zeros((16, 256), dtype=torch.bfloat16, device=cuda)
    assert ops.moe_layer_w4(x, router, bank, 4).shape == (0, 256)
    assert fused_moe_forward_w4(x, torch.zeros(17, dtype=torch.int64, device=cuda), bank).shape == (0, 256)


def test_bad_expert_ids_are_reported(cuda):
    p = ref.parts(4, 256, 128, 64, False, device=cuda)
    bank = bank_of(p)
    x = rows(3, 256, 1, cuda)
    ids = torch.tensor([[0, 1], [2, 9], [-1, 3]], dtype=torch.int32, device=cuda)
    y = ops.experts_w4(x, ids, torch.ones((3, 2), device=cuda), bank)
    with pytest.raises(ops.MoEKernelError, match="expert id"):
        ops.check_status(cuda)
    ids2 = torch.tensor([[0, 1], [2, 2], [3, 3]], dtype=torch.int32, device=cuda)
    w2 = torch.tensor([[1.0, 1.0], [1.0, 0.0], [0.0, 1.0]], device=cuda)
    want, bound = ref.experts(p, x, ids2, w2)
    close(y, want, bound)  # the good records are computed
    ops.check_status(cuda)


def test_non_finite_activations_stay_in_their_token(cuda):
    E, H, I, k, T = 8, 256, 128, 2, 20
    p = ref.parts(E, H, I, 64, False, device=cuda)
    bank = bank_of(p)
    gen = torch.Generator().manual_seed(1)
    ids = torch.rand((T, E), generator=gen).argsort(1)[:, :k].int().contiguous().to(cuda)
    w = torch.rand((T, k), generator=gen).to(cuda)
    x = rows(T, H, 2, cuda)
    clean = ops.experts_w4(x, ids, w, bank)
    x[5, 17] = float("nan")
    x[6, 3] = float("inf")
    y = ops.experts_w4(x, ids, w, bank)
    ops.check_status(cuda)
    keep = torch.ones(T, dtype=torch.bool, device=cuda)
    keep[5] = keep[6] = False
    assert torch.equal(y[keep], clean[keep])
    assert bool(y[5].isnan().all()) and not bool(torch.isfinite(y[6]).any())


def test_given_workspace_and_graph(cuda):
    """A captured call replays on new inputs; workspaces of the queried size suffice."""
    E, H, I, k, T = 32, 512, 128, 4, 6
    p = ref.parts(E, H, I, 64, False, device=cuda)
    bank = bank_of(p)
    router = (torch.randn((E, H), generator=torch.Generator().manual_seed(1)) * 0.08).bfloat16().to(cuda)
    for T in (6, 200):
        x = rows(T, H, 3, cuda)
        out = torch.empty_like(x)
        ws = torch.empty(ops.moe_layer_w4_workspace_bytes(T, k, bank), dtype=torch.uint8, device=cuda)
        ops.moe_layer_w4(x, router, bank, k, out=out, workspace=ws)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            ops.moe_layer_w4(x, router, bank, k, out=out, workspace=ws)
        for seed in (11, 12):
            x.copy_(rows(T, H, seed, cuda))
            graph.replay()
            got = out.clone()
            assert torch.equal(got, ops.moe_layer_w4(x, router, bank, k))
    ops.check_status(cuda)


def test_two_streams_at_once(cuda):
    E, H, I, k, T = 32, 512, 128, 4, 5
    p = ref.parts(E, H, I, 64, False, device=cuda)
    bank = bank_of(p)
    router = (torch.randn((E, H), generator=torch.Generator().manual_seed(1)) * 0.08).bfloat16().to(cuda)
    xs = [rows(T, H, s, cuda) for s in range(4)]
    want = [ops.moe_layer_w4(x, router, bank, k) for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(cuda) for _ in xs]
    got = []
    for _ in range(10):
        got = []
        for x, s in zip(xs, streams):
            with torch.cuda.stream(s):
                got.append(ops.moe_layer_w4(x, router, bank, k))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    ops.check_status(cuda)


# ------------------------------------------------------------------ block norm


@pytest.mark.parametrize("T,H", [(1, 8), (1, 2048), (3, 264), (17, 2048), (5, 5120), (2, 16392), (1500, 264),
                                 (2048, 5120), (2100, 8192), (8200, 1032), (1100, 4104),
                                 (1030, 2056), (8192, 2048),
                                 (1, 32768), (1000, 1024)])
@pytest.mark.parametrize("gate,act", [("absent", "none"), ("token", "sigmoid"), ("channel", "none"),
                                      ("element", "tanh"), ("channel", "sigmoid"), ("element", "none")])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_block_norm(cuda, T, H, gate, act, dtype):
    gen = torch.Generator().manual_seed(T + H)
    x = (torch.randn((T, H), generator=gen) * 2).bfloat16().to(cuda)
    d = (torch.randn((T, H), generator=gen) * 0.5).bfloat16().to(cuda)
    post, pre = ((torch.randn(H, generator=gen) * 0.2 + 1).to(cuda) for _ in range(2))
    shape = {"absent": None, "token": (T, 1), "channel": (H,), "element": (T, H)}[gate]
    g = None if shape is None else torch.randn(shape, generator=gen).to(dtype).to(cuda)
    h, y = ops.block_norm(x, d, post, pre, 1e-6, gate=g, gate_act=act, residual_scale=0.7)
    wh, wy, bh, by = ref.block_norm(x, d, post, pre, 1e-6, g, act, 0.7)
    close(h, wh, bh, "h")
    close(y, wy, by, "y")


def test_block_norm_rows_of_zeros_and_shapes(cuda):
    H = 256
    post, pre = torch.ones(H, device=cuda), torch.ones(H, device=cuda)
    x = rows(6, H, 1, cuda).view(2, 3, H)
    d = torch.zeros_like(x)
    h, y = ops.block_norm(x, d, post, pre, 1e-6)
    assert torch.equal(h, x) and y.shape == x.shape
    z = torch.zeros_like(x)
    h, y = ops.block_norm(z, z, post, pre, 1e-6)
    assert not bool(h.any()) and not bool(y.any())
    d[1, 2, 5] = float("nan")
    h, y = ops.block_norm(x, d, post, pre, 1e-6)
    assert bool(h[1, 2].isnan().all()) and bool(torch.isfinite(h[0].float()).all())
    e = torch.empty((0, H), dtype=torch.bfloat16, device=cuda)
    assert ops.block_norm(e, e, post, pre, 1e-6)[0].shape == (0, H)


def test_block_norm_equals_add_rmsnorm_up_to_rounding(cuda):
    """With unit post weight and a delta of unit mean square, h is x + delta."""
    T, H = 9, 512
    x = rows(T, H, 1, cuda)
    d = torch.where(rows(T, H, 2, cuda) > 0, 1.0, -1.0).bfloat16()
    one, pre = torch.ones(H, device=cuda), torch.rand(H, device=cuda) + 0.5
    h, y = ops.block_norm(x, d, one, pre, 0.0)
    h2, y2 = ops.add_rmsnorm(x, pre, 0.0, delta=d)
    assert (h.float() - h2.float()).abs().max() <= 2 * ref.BF16 * h2.float().abs().max()
    assert ((y.float() - y2.float()).norm() / y2.float().norm()) <= 2 * ref.BF16
