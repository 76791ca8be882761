"""``PermutedSparseMoE`` — drop-in for C5/python/solution.py:82-161.

Same constructor, attributes (``gate``, ``experts[e].{gate,up,down}_proj``)
and forward contract (``[..., H] -> same shape``).  The forward is one C-ABI
call, ``moe_layer_forward``: router + top-k on tcgen05, a stable counting
sort, the row gather, the w13 grouped GEMM with SwiGLU fused, the w2 grouped
GEMM with the top-k weight fused, and a deterministic k-way combine.  It
issues no host synchronisation (the reference syncs once per expert on
``.item()``, C5:144).  The keyword extra ``index_add="atomic"`` switches the
un-permute to the reference's own semantics (index_add_, C5:160: fp32 atomic
accumulation per token, fused into the down GEMM).  With the keyword extra
``check_errors=True`` every forward synchronises and raises
``ops.MoEKernelError`` if a kernel reported a failure in the device status
word; by default the forward never synchronises and a failure is only
recorded there (``ops.check_status`` reads it).  With the keyword extra
``decode_weights=True`` the module also keeps the down weights transposed
(one more copy of ``w_down``) and runs batches of up to 4 tokens on the
one-pass decode layer.  With the keyword extra
``expert_weights="w4"`` the forward runs on a 4-bit copy of the expert weights
(``ops.moe_layer_w4``; groups of ``group_size`` columns, with zero points unless
``symmetric``), rounded on first use.  Both copies are made again by the next
forward after the weights were written: through the stacked tensors, through an
expert's parameters (``load_state_dict``, an optimizer's step) or by re-binding.
Only writes that autograd's version counters do not see (through ``.data``, or
by a kernel on the raw pointer) need ``down_weights_transposed(refresh=True)``
or ``experts_4bit(refresh=True)``.  A copy is made again in its place in memory,
for graphs that captured a forward; a replay itself does not look for writes.

The module must be bf16 on a CUDA device: there is no CPU path.
"""

from __future__ import annotations

import operator

import torch
from torch import nn

from . import ops
from .experts import ExpertBank, SwiGLU_MLP, router_bias_of
from .w4 import BLOCK, GROUPS, MAX_COLUMNS, W4Experts

__all__ = ["PermutedSparseMoE", "SwiGLU_MLP"]

_version_of = operator.attrgetter("_version")


class _Source:
    """The weights that a copy in another form was made from, as they were then: the
    stacked tensors themselves (held, so that no later stack lies in their place and
    passes for them) and how often these and the experts' parameters had been written.
    The parameters are views of the stacks with version counters of their own, which
    only grow, so the sum stays the same only if none was written.  Reading the 384
    counters of 128 experts takes the host about 15 us."""

    def __init__(self, stacks, params) -> None:
        self.stacks = tuple(stacks)
        self._written = self.stacks + tuple(params)
        self._writes = self._count()

    def _count(self) -> int:
        return sum(map(_version_of, self._written))

    def unchanged(self, stacks) -> bool:
        return all(map(operator.is_, self.stacks, stacks)) and self._count() == self._writes

    def unlike(self, stacks) -> bool:
        """Whether a copy of these would not fit where the one of those lies."""
        return any((a.shape, a.dtype, a.device) != (b.shape, b.dtype, b.device)
                   for a, b in zip(self.stacks, stacks))


class PermutedSparseMoE(nn.Module):
    """Single-GPU sparse MoE with permutation + grouped compute (C5:82-161)."""

    def __init__(self, hidden: int, intermediate: int, num_experts: int, top_k: int,
                 norm_topk_prob: bool = True, *, index_add: str = "deterministic",
                 check_errors: bool = False, decode_weights: bool = False,
                 expert_weights: str = "bf16", group_size: int = 128,
                 symmetric: bool = True) -> None:
        super().__init__()
        ops._combine_mode(index_add)  # validate
        if expert_weights not in ("bf16", "w4"):
            raise ValueError(f'expert_weights must be "bf16" or "w4", got {expert_weights!r}')
        if expert_weights == "w4":
            if index_add != "deterministic" or decode_weights:
                raise ValueError('expert_weights="w4" has the deterministic combine and a decode '
                                 "layer of its own: no index_add, no decode_weights")
            if group_size not in GROUPS or hidden % group_size or intermediate % group_size:
                raise ValueError(f"group_size must be one of {GROUPS} and divide hidden and "
                                 f"intermediate, got {group_size}")
            for name, n in (("hidden", hidden), ("intermediate", intermediate)):
                if n % BLOCK or n > MAX_COLUMNS:
                    raise ValueError(f"4-bit experts need {name} to be a multiple of {BLOCK}, at "
                                     f"most {MAX_COLUMNS}, got {n}")
        self.expert_weights = expert_weights
        self.group_size = group_size
        self.symmetric = symmetric
        self._w4 = None
        self._w4_source = None
        self.index_add = index_add
        self.check_errors = check_errors
        self.decode_weights = decode_weights
        self._w_down_t = None
        self._w_down_t_source = None
        self.hidden = hidden
        self.intermediate = intermediate
        self.num_experts = num_experts
        self.top_k = top_k
        self.norm_topk_prob = norm_topk_prob
        self.gate = nn.Linear(hidden, num_experts, bias=False)
        self.experts = nn.ModuleList(SwiGLU_MLP(hidden, intermediate) for _ in range(num_experts))
        self._bank = ExpertBank()

    def __getstate__(self):
        """A copy of the module makes its own forms of its weights, on first use."""
        return {**self.__dict__, "_w4": None, "_w4_source": None, "_w_down_t": None,
                "_w_down_t_source": None}

    def _apply(self, fn, *args, **kwargs):
        self._bank.invalidate()
        self._w_down_t = self._w_down_t_source = None
        self._w4 = self._w4_source = None
        return super()._apply(fn, *args, **kwargs)

    def _parameters_of(self, **stacks):
        """The experts' parameters that are views of these stacked tensors, by projection.
        One that was made under inference mode has no version counter, so a parameter
        that has takes its place, on the same memory."""
        params = []
        with torch.inference_mode(False), torch.no_grad():
            for name, stack in stacks.items():
                for e, ex in enumerate(self.experts):
                    proj = getattr(ex, name)
                    try:
                        proj.weight._version
                    except RuntimeError:
                        proj.weight = nn.Parameter(stack[e], proj.weight.requires_grad)
                    params.append(proj.weight)
        return params

    def pack(self):
        """Stacked expert weights (w_gate, w_up, w_down), binding the per-expert
        parameters to views of them on first use, and anew after one was replaced."""
        return self._bank.bind(self.experts)

    def down_weights_transposed(self, refresh: bool = False) -> torch.Tensor:
        """w_down as [E, I, H] for the one-pass decode layer: built on first
        use and rebuilt when the down weights are re-bound or written in place,
        through the stacked tensor or an expert's parameter.  Writes through
        ``experts[e].down_proj.weight.data`` leave no trace: call with
        ``refresh=True`` after those.  It is rebuilt in its place, so a graph that
        captured a forward reads the new weights once this (or the module) was
        called; until the module is moved or cast, which ends such a graph."""
        wd = self._bank.bind(self.experts, every=refresh)[2]
        if refresh or self._w_down_t is None or not self._w_down_t_source.unchanged((wd,)):
            if wd.is_cuda and torch.cuda.is_current_stream_capturing():
                return ops.transpose_down_weights(wd)  # recorded, not done: not kept
            source = _Source((wd,), self._parameters_of(down_proj=wd))
            with torch.inference_mode(False), torch.no_grad():
                if self._w_down_t is None or self._w_down_t_source.unlike((wd,)):
                    self._w_down_t = ops.transpose_down_weights(wd)
                else:
                    self._w_down_t.copy_(wd.transpose(1, 2))
            self._w_down_t_source = source
        return self._w_down_t

    def experts_4bit(self, refresh: bool = False) -> W4Experts:
        """The 4-bit bank of ``expert_weights="w4"``, rebuilt under the same rules as
        ``down_weights_transposed``, for all three projections.  Building it
        synchronises, so call this (or the module) once before a graph capture."""
        weights = self._bank.bind(self.experts, every=refresh)
        if refresh or self._w4 is None or not self._w4_source.unchanged(weights):
            gate, up, down = weights
            source = _Source(weights, self._parameters_of(gate_proj=gate, up_proj=up,
                                                          down_proj=down))
            self._w4 = W4Experts.quantize(*weights, self.group_size, self.symmetric,
                                          into=self._w4)
            self._w4_source = source
        return self._w4

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        shape = x.shape
        x_flat = x.reshape(-1, shape[-1])
        if not x_flat.is_contiguous():
            x_flat = x_flat.contiguous()
        if self.expert_weights == "w4":
            y = ops.moe_layer_w4(x_flat, self.gate.weight, self.experts_4bit(), self.top_k,
                                 self.norm_topk_prob, bias=router_bias_of(self.gate))
        else:
            wg, wu, wd = self._bank.bind(self.experts, every=False)
            w_down_t = None
            if self.decode_weights and 0 < x_flat.shape[0] <= 4:
                w_down_t = self.down_weights_transposed()
            y = ops.moe_layer(x_flat, self.gate.weight, wg, wu, wd, self.top_k,
                              self.norm_topk_prob, bias=router_bias_of(self.gate),
                              index_add=self.index_add, w_down_t=w_down_t)
        if self.check_errors:
            ops.check_status(y.device)
        return y.reshape(shape)
