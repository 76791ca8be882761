"""The operators of the 4-bit expert path and the block's norm, as cases to be measured.

Kinds of case:

* ``layer``    the whole mixture-of-experts layer for a few tokens (router, top-k, 4-bit experts, combine)
* ``experts``  the 4-bit experts for tokens whose routing is given (a local shard of them included)
* ``grouped``  the 4-bit experts for rows that are sorted by expert already, unweighted
* ``norm``     the norm after a block, its gate and residual scale, and the norm before the next block

4-bit weights: ``w[n, c] = scale[n, c // group] * (code[n, c] - zero[n, c // group])`` with codes of 0..15
and zero points of 0..15 (8 throughout where a case has none of its own).
"""

import math

import torch

own = False

FULL = {"hidden": 2048, "intermediate": 768, "experts": 128, "top_k": 8}


def listed():
    return [
        # one token of one request: the latency of a decode step
        {"name": "layer 1 token", "kind": "layer", "tokens": 1, **FULL, "group": 128, "zeros": False, "bias": False, "norm": True},
        # a few requests decoded together; a router with a bias, zero points, weights of the softmax over all experts
        {"name": "layer 7 tokens", "kind": "layer", "tokens": 7, **FULL, "group": 64, "zeros": True, "bias": True, "norm": False},
        # a decode batch: most experts see one record or two
        {"name": "experts 24 tokens", "kind": "experts", "tokens": 24, **FULL, "local": 128, "first": 0, "skew": 0.0, "group": 128, "zeros": False},
        # a large decode batch: every expert is read, for sixteen records each
        {"name": "experts 256 tokens", "kind": "experts", "tokens": 256, **FULL, "local": 128, "first": 0, "skew": 0.3, "group": 128, "zeros": False},
        # one rank's quarter of the experts under skewed routing: tokens without any local expert, experts without tokens
        {"name": "experts 1001 tokens shard", "kind": "experts", "tokens": 1001, **FULL, "local": 32, "first": 64, "skew": 0.8, "group": 32, "zeros": True},
        # a prompt batch
        {"name": "experts 8192 tokens", "kind": "experts", "tokens": 8192, **FULL, "local": 128, "first": 0, "skew": 0.2, "group": 128, "zeros": False},
        # rows another step has sorted, ragged, with empty experts
        {"name": "grouped 77 rows", "kind": "grouped", "rows": 77, "hidden": 2048, "intermediate": 768, "experts": 128, "skew": 0.8, "group": 64, "zeros": False},
        # the same for a prompt, on a rank that holds half of each expert's columns
        {"name": "grouped 6000 rows", "kind": "grouped", "rows": 6000, "hidden": 2048, "intermediate": 384, "experts": 64, "skew": 0.4, "group": 128, "zeros": True},
        # between two blocks, one token: a gate for each channel
        {"name": "norm 1 token", "kind": "norm", "tokens": 1, "hidden": 2048, "gate": "channel", "act": "none", "scale": 0.5},
        # a decode batch: a sigmoid gate for each token
        {"name": "norm 333 tokens", "kind": "norm", "tokens": 333, "hidden": 2048, "gate": "token", "act": "sigmoid", "scale": 1.0},
        # a prompt batch: a gate for each channel
        {"name": "norm 16384 tokens", "kind": "norm", "tokens": 16384, "hidden": 2048, "gate": "channel", "act": "none", "scale": 0.5},
        # a prompt batch of a wide model: a gate of its own for every element
        {"name": "norm 9001 tokens wide", "kind": "norm", "tokens": 9001, "hidden": 5120, "gate": "element", "act": "tanh", "scale": 0.7},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["layer", "experts", "experts", "grouped", "norm"])
    if kind == "norm":
        hidden = 8 * _log_int(rng, 8, 1024)
        most = min(32768, 9001 * 5120 // hidden)
        return {"kind": kind, "tokens": _log_int(rng, 1, most), "hidden": hidden, "gate": rng.choice(["absent", "token", "channel", "element"]),
                "act": rng.choice(["none", "sigmoid", "tanh"]), "scale": rng.choice([1.0, 0.5, 0.22])}
    group = rng.choice([32, 64, 128])
    step = max(group, 64)
    hidden, inner = step * rng.randint(512 // step, 4096 // step), step * _log_int(rng, 1, 1536 // step)
    zeros = rng.random() < 0.5
    most = 3 * 2048 * 768 * 128  # no more weights than the listed cases have
    if kind == "layer":
        experts = rng.choice([e for e in (16, 32, 64, 128, 256) if 3 * hidden * inner * e <= most])
        return {"kind": kind, "tokens": _log_int(rng, 1, 64), "hidden": hidden, "intermediate": inner, "experts": experts, "top_k": rng.randint(1, 8),
                "group": group, "zeros": zeros, "bias": rng.random() < 0.3, "norm": rng.random() < 0.7}
    experts = max(8, min(_log_int(rng, 8, 256), most // (3 * hidden * inner)))
    if kind == "grouped":
        rows = _log_int(rng, 1, min(65536, 65536 * 2048 * 768 // (hidden * inner)))
        return {"kind": kind, "rows": rows, "hidden": hidden, "intermediate": inner, "experts": experts, "skew": rng.choice([0.0, 0.4, 0.8]), "group": group, "zeros": zeros}
    local = rng.choice([experts, experts, max(1, experts // 4)])
    top_k = rng.randint(1, 8)
    tokens = _log_int(rng, 1, min(8192, 65536 * 2048 * 768 // (hidden * inner * top_k)))
    return {"kind": kind, "tokens": tokens, "hidden": hidden, "intermediate": inner, "experts": experts, "top_k": top_k, "local": local,
            "first": rng.randint(0, experts - local), "skew": rng.choice([0.0, 0.3, 0.8]), "group": group, "zeros": zeros}


# ---------------------------------------------------------------------------------------------- inputs


def _matrix(gen, experts, rows, columns, group, zeros, std):
    """Codes, scales and zero points of stacked matrices whose values spread like trained weights of this deviation."""
    codes = torch.randn((experts, rows, columns), generator=gen, device="cuda").mul_(3.0).add_(8.0).round_().clamp_(0, 15).to(torch.uint8)
    shape = (experts, rows, columns // group)
    scales = (torch.rand(shape, generator=gen, device="cuda").add_(0.5) * (std / 3.0)).bfloat16()
    points = torch.randint(6, 11, shape, generator=gen, device="cuda", dtype=torch.uint8) if zeros else None
    return codes, scales, points


def _popularity(gen, experts, skew):
    """Log-odds of the experts: a power law over a random order of them."""
    order = torch.randperm(experts, generator=gen, device="cuda")
    return -skew * torch.log(order.float() + 1.0)


def _inputs(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    hidden = case["hidden"]
    if case["kind"] == "norm":
        tokens = case["tokens"]
        made = {name: torch.randn((tokens, hidden), generator=gen, device="cuda").mul_(scale).bfloat16() for name, scale in (("x", 2.0), ("delta", 0.6))}
        for name in ("post", "pre"):
            made[name] = torch.randn(hidden, generator=gen, device="cuda") * 0.2 + 1.0
        shape = {"absent": None, "token": (tokens, 1), "channel": (hidden,), "element": (tokens, hidden)}[case["gate"]]
        made["gate"] = None if shape is None else torch.randn(shape, generator=gen, device="cuda").mul_(0.5).add_(0.5).bfloat16()
        return made
    inner, experts, group, zeros = case["intermediate"], case["experts"], case["group"], case["zeros"]
    held = case.get("local", experts)
    made = {
        "w_gate": _matrix(gen, held, inner, hidden, group, zeros, hidden**-0.5),
        "w_up": _matrix(gen, held, inner, hidden, group, zeros, hidden**-0.5),
        "w_down": _matrix(gen, held, hidden, inner, group, zeros, inner**-0.5),
    }
    rows = case["rows"] if case["kind"] == "grouped" else case["tokens"]
    made["x"] = torch.randn((rows, hidden), generator=gen, device="cuda").bfloat16()
    if case["kind"] == "layer":
        made["router"] = (torch.randn((experts, hidden), generator=gen, device="cuda") * (1.8 * hidden**-0.5)).bfloat16()
        made["bias"] = torch.randn(experts, generator=gen, device="cuda") if case["bias"] else None
        return made
    odds = _popularity(gen, experts, case["skew"])
    picks = 1 if case["kind"] == "grouped" else case["top_k"]
    noise = -torch.log(-torch.log(torch.rand((rows, experts), generator=gen, device="cuda").clamp_(1e-7, 1 - 1e-7)))
    value, ids = torch.topk(odds + noise, picks, dim=1)
    if case["kind"] == "grouped":
        counts = torch.bincount(ids.reshape(-1), minlength=experts)
        made["offsets"] = torch.cat([counts.new_zeros(1), counts.cumsum(0)])
    else:
        made["ids"], made["weights"] = ids.int(), torch.softmax(value, 1)
    return made


def prepare(case, seed):
    state = {"case": case, **_inputs(case, seed)}
    if own and case["kind"] != "norm":
        from moe_inference_verify_microbench_b200 import W4Experts

        # the weights as a serving program keeps them: laid out once, when they are loaded
        state["bank"] = W4Experts.from_codes(state["w_gate"], state["w_up"], state["w_down"])
    return state


# ---------------------------------------------------------------------------------------------- the passes


def _run_own(s):
    from moe_inference_verify_microbench_b200 import fused_moe_forward_w4, ops

    case = s["case"]
    if case["kind"] == "layer":
        return ops.moe_layer_w4(s["x"], s["router"], s["bank"], case["top_k"], norm_topk_prob=case["norm"], bias=s["bias"])
    if case["kind"] == "experts":
        return ops.experts_w4(s["x"], s["ids"], s["weights"], s["bank"], num_experts=case["experts"], e_begin=case["first"])
    if case["kind"] == "grouped":
        return fused_moe_forward_w4(s["x"], s["offsets"], s["bank"])
    return ops.block_norm(s["x"], s["delta"], s["post"], s["pre"], 1e-6, gate=s["gate"], gate_act=case["act"], residual_scale=case["scale"])


def _values(matrix, group, active):
    """The weights of the active experts, [A, N, K] in 32 bits."""
    codes, scales, zeros = matrix
    codes, scales = codes[active], scales[active].float()
    wide = codes.float().view(*scales.shape, group)
    wide -= 8.0 if zeros is None else zeros[active].float().unsqueeze(-1)
    wide *= scales.unsqueeze(-1)
    return wide.view(codes.shape)


def _expert_rows(s, rows, owner):
    """The experts' products for 32-bit rows, each with the expert `owner` of the held ones: a padded batched product."""
    active, slot, counts = torch.unique(owner, return_inverse=True, return_counts=True)
    group = s["case"]["group"]
    order = torch.argsort(slot, stable=True)
    place = torch.arange(order.numel(), device=order.device) - (counts.cumsum(0) - counts)[slot[order]]
    padded = rows.new_zeros((active.numel(), int(counts.max()), rows.shape[1]))
    padded[slot[order], place] = rows[order]
    gate = padded @ _values(s["w_gate"], group, active).transpose(1, 2)
    up = padded @ _values(s["w_up"], group, active).transpose(1, 2)
    out = (gate / (1.0 + torch.exp(-gate)) * up) @ _values(s["w_down"], group, active).transpose(1, 2)
    back = torch.empty_like(rows)
    back[order] = out[slot[order], place]
    return back


def _weighted(s, ids, weights, first, held):
    """Each token's experts, weighted and summed; experts that are not held add nothing."""
    x, picks = s["x"], ids.shape[1]
    flat = ids.reshape(-1).long() - first
    slots = ((flat >= 0) & (flat < held)).nonzero().squeeze(1)
    result = x.new_zeros((flat.numel(), x.shape[1]), dtype=torch.float32)
    if slots.numel():
        result[slots] = _expert_rows(s, x.float()[slots // picks], flat[slots])
    return (result.view(*ids.shape, -1) * weights.unsqueeze(-1)).sum(1).bfloat16()


def _route(s):
    """Logits as the router defines them, rounded to bf16; the largest, the lowest expert among equal ones; their weights."""
    case = s["case"]
    logits = s["x"].float() @ s["router"].float().t()
    if s["bias"] is not None:
        logits = logits + s["bias"]
    logits = logits.bfloat16().float()
    value, ids = (part[:, : case["top_k"]] for part in torch.sort(logits, dim=1, descending=True, stable=True))
    over = value if case["norm"] else logits
    top = logits.amax(1, keepdim=True)
    return ids, torch.exp(value - top) / torch.exp(over - top).sum(1, keepdim=True)


def _gated(case, gate):
    gate = gate.float()
    if case["act"] == "sigmoid":
        return 1.0 / (1.0 + torch.exp(-gate))
    if case["act"] == "tanh":
        return 1.0 - 2.0 / (torch.exp(2.0 * gate) + 1.0)
    return gate


def _run_plain(s):
    case = s["case"]
    if case["kind"] == "layer":
        ids, weights = _route(s)
        return _weighted(s, ids, weights, 0, case["experts"])
    if case["kind"] == "experts":
        return _weighted(s, s["ids"], s["weights"], case["first"], case["local"])
    if case["kind"] == "grouped":
        owner = torch.repeat_interleave(torch.arange(case["experts"], device="cuda"), s["offsets"].diff())
        return _expert_rows(s, s["x"].float(), owner).bfloat16()
    delta = s["delta"].float()
    step = delta * torch.rsqrt((delta * delta).mean(1, keepdim=True) + 1e-6) * s["post"] * case["scale"]
    if s["gate"] is not None:
        step = step * _gated(case, s["gate"])
    h = s["x"].float() + step
    return h.bfloat16(), (h * torch.rsqrt((h * h).mean(1, keepdim=True) + 1e-6) * s["pre"]).bfloat16()


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---------------------------------------------------------------------------------------------- what a pass cannot do without


def work(case):
    hidden = case["hidden"]
    if case["kind"] == "norm":
        tokens = case["tokens"]
        gate = {"absent": 0, "token": tokens, "channel": hidden, "element": tokens * hidden}[case["gate"]]
        return {"bytes": 8 * tokens * hidden + 2 * gate + 8 * hidden, "flops": 14 * tokens * hidden}
    inner, experts, group = case["intermediate"], case["experts"], case["group"]
    matrix = 3 * hidden * inner
    per_expert = matrix // 2 + matrix // group * (3 if case["zeros"] else 2)
    if case["kind"] == "grouped":
        rows = case["rows"]
        active = experts * (1.0 - (1.0 - 1.0 / experts) ** rows)
        return {"bytes": int(active * per_expert) + 4 * rows * hidden + 8 * (experts + 1), "flops": 2 * rows * matrix}
    tokens, top_k = case["tokens"], case["top_k"]
    share = min(1.0, top_k / experts)
    held = case.get("local", experts)
    active = held * (1.0 - (1.0 - share) ** tokens)  # experts that uniform routing reaches
    records = tokens * share * held
    total = {"bytes": int(active * per_expert) + 4 * tokens * hidden, "flops": int(2 * records * matrix)}
    if case["kind"] == "layer":
        total["bytes"] += 2 * experts * hidden
        total["flops"] += 2 * tokens * experts * hidden
    else:
        total["bytes"] += 8 * tokens * top_k
    return total


# ---------------------------------------------------------------------------------------------- in 64 bits


def _one(matrix, expert, group):
    codes, scales, zeros = matrix
    step = scales[expert].double().repeat_interleave(group, dim=1)
    point = 8.0 if zeros is None else zeros[expert].double().repeat_interleave(group, dim=1)
    return step * (codes[expert].double() - point)


def _mlp(made, expert, group, rows):
    g = rows @ _one(made["w_gate"], expert, group).t()
    u = rows @ _one(made["w_up"], expert, group).t()
    return (g * torch.sigmoid(g) * u) @ _one(made["w_down"], expert, group).t()


def exact(case, seed):
    made = _inputs(case, seed)
    x = made["x"].double()
    if case["kind"] == "norm":
        delta = made["delta"].double()
        n = delta / (delta.pow(2).mean(-1, keepdim=True) + 1e-6).sqrt() * made["post"].double()
        if made["gate"] is not None:
            gate = made["gate"].double()
            n = n * {"none": lambda v: v, "sigmoid": torch.sigmoid, "tanh": torch.tanh}[case["act"]](gate)
        h = x + case["scale"] * n
        return h, h / (h.pow(2).mean(-1, keepdim=True) + 1e-6).sqrt() * made["pre"].double()
    group = case["group"]
    y = torch.zeros_like(x)
    if case["kind"] == "grouped":
        ends = made["offsets"].tolist()
        for expert in range(case["experts"]):
            first, last = ends[expert], ends[expert + 1]
            if last > first:
                y[first:last] = _mlp(made, expert, group, x[first:last])
        return y
    if case["kind"] == "layer":
        logits = x @ made["router"].double().t()
        if made["bias"] is not None:
            logits = logits + made["bias"].double()
        logits = logits.bfloat16().double()  # the router's logits are bf16 by definition
        spread = torch.softmax(logits, 1)
        ids = torch.argsort(logits, dim=1, descending=True, stable=True)[:, : case["top_k"]]
        weights = spread.gather(1, ids)
        if case["norm"]:
            weights = weights / weights.sum(1, keepdim=True)
        first, held = 0, case["experts"]
    else:
        ids, weights, first, held = made["ids"].long(), made["weights"].double(), case["first"], case["local"]
    for expert in range(held):
        token, place = (ids == first + expert).nonzero(as_tuple=True)
        if token.numel():
            y.index_add_(0, token, weights[token, place].unsqueeze(1) * _mlp(made, expert, group, x[token]))
    return y
