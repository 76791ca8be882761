"""Plain 64-bit forms of the 4-bit expert operators and the block norm."""

from __future__ import annotations

import torch

BF16 = torch.finfo(torch.bfloat16).eps / 2  # a rounding to bf16 is off by at most this, relatively


def matrix(gen, E, N, K, group, zeros, std, device):
    """Random (codes, scales, zero points)."""
    codes = (torch.randn((E, N, K), generator=gen) * 3 + 8).round().clamp(0, 15).to(torch.uint8)
    shape = (E, N, K // group)
    scales = ((torch.rand(shape, generator=gen) + 0.5) * (std / 3)).bfloat16()
    z = torch.randint(0, 16, shape, generator=gen, dtype=torch.uint8) if zeros else None
    return (codes.to(device), scales.to(device), None if z is None else z.to(device))


def parts(E, H, I, group, zeros, seed=0, device="cpu"):
    gen = torch.Generator().manual_seed(seed)
    return (matrix(gen, E, I, H, group, zeros, H ** -0.5, device),
            matrix(gen, E, I, H, group, zeros, H ** -0.5, device),
            matrix(gen, E, H, I, group, zeros, I ** -0.5, device))


def values(m):
    """The weights in 64 bits, [E, N, K]."""
    codes, scales, zeros = m
    g = codes.shape[-1] // scales.shape[-1]
    q = codes.double().reshape(*scales.shape, g)
    q = q - (8.0 if zeros is None else zeros.double().unsqueeze(-1))
    return (q * scales.double().unsqueeze(-1)).reshape(codes.shape)


def operand_sums(m, x, e):
    """sum_k s * 144 * |x_k| per (row of x, output): what the fp32 sums of products
    with 128 + q are formed from, in absolute value."""
    codes, scales, _ = m
    g = codes.shape[-1] // scales.shape[-1]
    wide = scales[e].double().abs().repeat_interleave(g, dim=1) * 144.0
    return x.double().abs() @ wide.t()


# A group is summed by eight matrix instructions at most, each adding 17 numbers that
# are off by at most 2^-24 of the largest: 8 * 17 * 2^-24 < 2^-16 of the absolute sum,
# which also covers the few fp32 additions of groups and warps.
ACC = 2.0 ** -16


def weight_rounding(values, x):
    """sum_k BF16 * |w_k x_k|: what rounding every weight to bf16 can move a product by.
    The tensor-memory form for many records per expert (records >= TC_RECORDS * experts)
    does that; the streaming form keeps the weights exact."""
    return BF16 * (x.double().abs() @ values.abs().t())


TC_RECORDS = 8


def swiglu_rows(w_gate, w_up, vg, vu, x, e, rounded):
    """h = silu(x Wg^T) * (x Wu^T) of expert e in 64 bits, and a bound of a
    kernel's error: the rounding of h, the fp32 sums and, if so, of the weights."""
    xd = x.double()
    g, u = xd @ vg[e].t(), xd @ vu[e].t()
    dg, du = ACC * operand_sums(w_gate, x, e), ACC * operand_sums(w_up, x, e)
    if rounded:
        dg, du = dg + weight_rounding(vg[e], x), du + weight_rounding(vu[e], x)
    sg = torch.sigmoid(g)
    # |silu'| <= 1.1, |silu(g)| <= |g|; the fast exponential and division: 2^-20 relative
    h = g * sg * u
    bound = BF16 * h.abs() + 1.1 * dg * (u.abs() + du) + (g * sg).abs() * du + 2.0 ** -20 * h.abs()
    return h, bound * 1.01 + 1e-30


def down_rows(w_down, vd, h, e, rounded):
    """o = h Wd^T of expert e in 64 bits, and the bound of its sums."""
    do = ACC * operand_sums(w_down, h, e)
    return h.double() @ vd[e].t(), do + weight_rounding(vd[e], h) if rounded else do


def experts(p, x, ids, weights, e_begin=0, num_experts=None):
    """y = sum_j w_j MLP_{ids_j}(x) in 64 bits, and a bound of a kernel's error that
    rounds h, each weighted row and y to bf16, and the weights where the records are many."""
    vg, vu, vd = (values(m) for m in p)
    T, H = x.shape
    rounded = ids.numel() // (num_experts or vg.shape[0]) >= TC_RECORDS
    y = torch.zeros((T, H), dtype=torch.float64, device=x.device)
    bound = torch.zeros_like(y)
    for e in range(vg.shape[0]):
        n, j = (ids == e_begin + e).nonzero(as_tuple=True)
        if not n.numel():
            continue
        w = weights[n, j].double().unsqueeze(1)
        h, dh = swiglu_rows(p[0], p[1], vg, vu, x[n], e, rounded)
        o, do = down_rows(p[2], vd, h, e, rounded)
        do = do * 1.01 + dh @ vd[e].abs().t() * (1 + BF16)
        y.index_add_(0, n, w * o)
        bound.index_add_(0, n, w.abs() * (do + BF16 * (o.abs() + do)))
    return y, bound + BF16 * (y.abs() + bound) + 1e-30


def roundings(parts, rounded):
    """Independent roundings that the relative error of a result is made of: the given
    ones, and of the weights of the gate and up products (through silu, whose slope
    is at most 1.1) and of the down product."""
    more = {"h": 2.5, "out": 1.0, "y": 3.5}[parts] if rounded else 0.0
    return {"h": 1, "out": 1, "y": 3}[parts] + more


def route(x, router, bias, k, norm):
    """bf16 logits, top-k (value descending, lower id first), weights."""
    logits = x.double() @ router.double().t()
    if bias is not None:
        logits = logits + bias.double()
    logits = logits.bfloat16().double()
    ids = torch.argsort(logits, dim=1, descending=True, stable=True)[:, :k]
    w = torch.softmax(logits, 1).gather(1, ids)
    return ids, w / w.sum(1, keepdim=True) if norm else w


def block_norm(x, delta, post, pre, eps, gate, act, scale):
    x, d = x.double(), delta.double()
    n = d / (d.pow(2).mean(-1, keepdim=True) + eps).sqrt() * post.double()
    if gate is not None:
        f = {"none": lambda v: v, "sigmoid": torch.sigmoid, "tanh": torch.tanh}[act]
        n = n * f(gate.double())
    h = x + scale * n
    y = h / (h.pow(2).mean(-1, keepdim=True) + eps).sqrt() * pre.double()
    # fp32 work on the row: a few dozen operations, each 2^-24 of its largest operand
    dh = BF16 * h.abs() + 2.0 ** -19 * (x.abs() + (scale * n).abs())
    dy = BF16 * y.abs() + 2.0 ** -18 * (y.abs() + (x.abs() + (scale * n).abs()) * pre.double().abs()
                                        / (h.pow(2).mean(-1, keepdim=True) + eps).sqrt())
    return h, y, dh + 1e-30, dy + 1e-30
