"""C8 drop-ins: ``HybridMoE`` (the hot path, in ``ep``) and ``HybridBlock``
(C8/python/solution.py:235-325), the pre-norm decoder block
``h = x + attn(norm(x)); y = h + moe(norm(h))`` that hosts it.

The attention and RMSNorm here are a plain PyTorch harness with the
reference's interfaces (C4 ``TPGQA``, C4/python/solution.py:169-276, and the
``RMSNorm(hidden, eps)`` that C8 imports): GQA with tensor-parallel heads,
KV-head replication when tp > n_kv_heads (C4:127), RoPE, causal SDPA and a
row-parallel output projection closed by an all_reduce on the TP group
(C1/python/solution.py:142).  They are not part of the optimised path.
``HybridBlock.forward`` runs the two RMSNorms and the first residual add in
one row kernel (``ops.add_rmsnorm``); the ``RMSNorm`` module keeps the
harness's PyTorch definition of the math.  With ``post_norm=True`` each branch's
output is normed too, gated and scaled before it is added, and the add, both
norms and the gate are one row kernel (``ops.block_norm``).
"""

from __future__ import annotations

import torch
import torch.distributed as dist
import torch.nn.functional as F
from torch import nn

from . import ops
from .ep import HybridMoE

__all__ = ["HybridMoE", "HybridBlock", "RMSNorm", "TPGQA"]


class RMSNorm(nn.Module):
    def __init__(self, hidden: int, eps: float = 1e-6) -> None:
        super().__init__()
        self.eps = eps
        self.weight = nn.Parameter(torch.ones(hidden))

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        xf = x.float()
        xf = xf * torch.rsqrt(xf.pow(2).mean(-1, keepdim=True) + self.eps)
        return (xf * self.weight.float()).to(x.dtype)


def _rope(x: torch.Tensor, base: float) -> torch.Tensor:
    """Rotate-half RoPE on [B, T, heads, d]."""
    T, d = x.shape[1], x.shape[-1]
    inv = 1.0 / (base ** (torch.arange(0, d, 2, device=x.device, dtype=torch.float32) / d))
    f = torch.outer(torch.arange(T, device=x.device, dtype=torch.float32), inv)
    cos = torch.cat([f, f], -1).cos()[None, :, None, :]
    sin = torch.cat([f, f], -1).sin()[None, :, None, :]
    x1, x2 = x[..., : d // 2], x[..., d // 2:]
    rot = torch.cat([-x2, x1], -1)
    return (x.float() * cos + rot.float() * sin).to(x.dtype)


class _ShardLoader(nn.Module):
    """Holds one rank's shard and copies it out of the full weight."""

    def __init__(self, weight: torch.Tensor, loader) -> None:
        super().__init__()
        self.weight = nn.Parameter(weight)
        self._loader = loader

    @torch.no_grad()
    def weight_loader(self, full_weight: torch.Tensor, shard_id: str | None = None) -> None:
        self._loader(self.weight, full_weight, shard_id)


class TPGQA(nn.Module):
    """Tensor-parallel grouped-query attention with KV replication."""

    def __init__(self, hidden: int, n_heads: int, n_kv_heads: int, head_dim: int,
                 rope_base: float = 10000.0, tp_size: int = 1, tp_rank: int = 0,
                 group: dist.ProcessGroup | None = None) -> None:
        super().__init__()
        assert n_heads % tp_size == 0
        self.hidden, self.head_dim, self.rope_base = hidden, head_dim, rope_base
        self.tp_size, self.tp_rank, self.group = tp_size, tp_rank, group
        self.q_per_rank = n_heads // tp_size
        self.kv_per_rank = max(1, n_kv_heads // tp_size)
        if tp_size > n_kv_heads:
            assert tp_size % n_kv_heads == 0
            self.kv_first = tp_rank // (tp_size // n_kv_heads)
        else:
            assert n_kv_heads % tp_size == 0
            self.kv_first = tp_rank * self.kv_per_rank
        qd, kvd = self.q_per_rank * head_dim, self.kv_per_rank * head_dim

        def load_qkv(w, full, shard_id):
            if shard_id == "q":
                w[:qd].copy_(full[tp_rank * qd:(tp_rank + 1) * qd])
            else:
                off = qd if shard_id == "k" else qd + kvd
                r0 = self.kv_first * head_dim
                w[off:off + kvd].copy_(full[r0:r0 + kvd])

        def load_o(w, full, _):
            w.copy_(full[:, tp_rank * qd:(tp_rank + 1) * qd])

        self.qkv_proj = _ShardLoader(torch.empty(qd + 2 * kvd, hidden), load_qkv)
        self.o_proj = _ShardLoader(torch.empty(hidden, qd), load_o)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        B, T, _ = x.shape
        d = self.head_dim
        qkv = F.linear(x, self.qkv_proj.weight)
        qd, kvd = self.q_per_rank * d, self.kv_per_rank * d
        q = qkv[..., :qd].reshape(B, T, self.q_per_rank, d)
        k = qkv[..., qd:qd + kvd].reshape(B, T, self.kv_per_rank, d)
        v = qkv[..., qd + kvd:].reshape(B, T, self.kv_per_rank, d)
        q, k = _rope(q, self.rope_base), _rope(k, self.rope_base)
        rep = self.q_per_rank // self.kv_per_rank
        k = k.repeat_interleave(rep, dim=2)
        v = v.repeat_interleave(rep, dim=2)
        o = F.scaled_dot_product_attention(q.transpose(1, 2), k.transpose(1, 2), v.transpose(1, 2),
                                           is_causal=True)
        o = o.transpose(1, 2).reshape(B, T, qd)
        out = F.linear(o, self.o_proj.weight)
        if self.tp_size > 1:
            dist.all_reduce(out, group=self.group)
        return out


class HybridBlock(nn.Module):
    """Pre-norm block under TP x DP x EP (C8/python/solution.py:235-325)."""

    def __init__(self, hidden: int, intermediate: int, n_heads: int, n_kv_heads: int,
                 head_dim: int, num_experts: int, top_k: int, tp_size: int, tp_rank: int,
                 tp_group: dist.ProcessGroup | None, ep_size: int, ep_rank: int,
                 ep_group: dist.ProcessGroup | None, norm_topk_prob: bool = True,
                 rope_base: float = 10000.0, rms_eps: float = 1e-6, *, post_norm: bool = False,
                 gate_act: str | None = None, residual_scale: float = 1.0,
                 **moe_options) -> None:
        """``moe_options``: keyword extras of ``HybridMoE`` (transport,
        max_tokens_per_rank, check_errors, overlap, exchange_sms).

        ``post_norm``: ``h = x + residual_scale * act(gate) * norm(attn(norm(x)))`` and the
        same around the experts, with norms of their own (``attn_post_norm``,
        ``moe_post_norm``).  ``gate_act`` ("none", "sigmoid" or "tanh") adds a learned
        gate per channel to each branch (``attn_gate``, ``moe_gate``); None: no gate."""
        super().__init__()
        if not post_norm and (gate_act is not None or residual_scale != 1.0):
            raise ValueError("gate_act and residual_scale need post_norm=True")
        if gate_act is not None:
            ops.check_gate_act(gate_act)
        self.post_norm = post_norm
        self.gate_act = gate_act
        self.residual_scale = residual_scale
        if post_norm:
            self.attn_post_norm = RMSNorm(hidden, eps=rms_eps)
            self.moe_post_norm = RMSNorm(hidden, eps=rms_eps)
            if gate_act is not None:
                self.attn_gate = nn.Parameter(torch.ones(hidden))
                self.moe_gate = nn.Parameter(torch.ones(hidden))
        self.attn_norm = RMSNorm(hidden, eps=rms_eps)
        self.attn = TPGQA(hidden, n_heads, n_kv_heads, head_dim, rope_base=rope_base,
                          tp_size=tp_size, tp_rank=tp_rank, group=tp_group)
        self.moe_norm = RMSNorm(hidden, eps=rms_eps)
        self.moe = HybridMoE(hidden, intermediate, num_experts, top_k, tp_size, tp_rank, tp_group,
                             ep_size, ep_rank, ep_group, norm_topk_prob, **moe_options)

    @torch.no_grad()
    def weight_loader(self, attn_norm_weight, q_weight, k_weight, v_weight, o_weight,
                      moe_norm_weight, gate_weight, expert_gate_weights, expert_up_weights,
                      expert_down_weights, *, attn_post_norm_weight=None,
                      moe_post_norm_weight=None, attn_gate=None, moe_gate=None) -> None:
        extras = []
        for have, name, given in (
                (self.post_norm, "attn_post_norm", attn_post_norm_weight),
                (self.post_norm, "moe_post_norm", moe_post_norm_weight),
                (self.gate_act is not None, "attn_gate", attn_gate),
                (self.gate_act is not None, "moe_gate", moe_gate)):
            if given is None:
                continue
            if not have:
                raise ValueError(f"this block has no {name}")
            own = getattr(self, name)
            extras.append((own.weight if isinstance(own, RMSNorm) else own, given))
        self.attn_norm.weight.data.copy_(attn_norm_weight)
        self.attn.qkv_proj.weight_loader(q_weight, "q")
        self.attn.qkv_proj.weight_loader(k_weight, "k")
        self.attn.qkv_proj.weight_loader(v_weight, "v")
        self.attn.o_proj.weight_loader(o_weight)
        self.moe_norm.weight.data.copy_(moe_norm_weight)
        self.moe.weight_loader(gate_weight, expert_gate_weights, expert_up_weights,
                               expert_down_weights)
        for own, given in extras:
            own.data.copy_(given)

    def _join(self, x, branch, post: RMSNorm, gate, pre: RMSNorm):
        """(x + scale * act(gate) * post(branch), its pre norm), one row kernel."""
        return ops.block_norm(x, branch.contiguous(), post.weight, pre.weight, pre.eps, gate=gate,
                              gate_act=self.gate_act or "none",
                              residual_scale=self.residual_scale)

    def forward(self, x: torch.Tensor, normed: torch.Tensor | None = None,
                next_norm: RMSNorm | None = None):
        """The block's output; with ``next_norm`` (the ``attn_norm`` of the block that
        follows) also that norm of it, taken in the kernel that makes the output, to be
        passed to that block as ``normed``."""
        # h = x + attn(norm(x)); y = h + moe(norm(h)) (C8:318-325).  Both norms
        # and the first residual add run in the fused row kernel.
        x = x.contiguous()
        if next_norm is not None and next_norm.eps != self.attn_norm.eps:
            raise ValueError(f"next_norm has eps {next_norm.eps}, this block {self.attn_norm.eps}")
        if normed is None:
            normed = ops.add_rmsnorm(x, self.attn_norm.weight, self.attn_norm.eps)
        elif normed.shape != x.shape:
            raise ValueError(f"normed must have the shape of x, got {tuple(normed.shape)}")
        a = self.attn(normed)
        if not self.post_norm:
            h, n2 = ops.add_rmsnorm(x, self.moe_norm.weight, self.moe_norm.eps,
                                    delta=a.contiguous())
            m = self.moe(n2)
            if next_norm is None:
                return h + m
            return ops.add_rmsnorm(h, next_norm.weight, next_norm.eps, delta=m.contiguous())
        gated = self.gate_act is not None
        h, n2 = self._join(x, a, self.attn_post_norm, self.attn_gate if gated else None,
                           self.moe_norm)
        y, n = self._join(h, self.moe(n2), self.moe_post_norm, self.moe_gate if gated else None,
                          self.attn_norm if next_norm is None else next_norm)
        return y if next_norm is None else (y, n)
