"""``fused_moe_forward`` — drop-in for C9/python/solution.py:207-222.

Same arguments and result: per expert e, rows ``offsets[e]:offsets[e+1]`` of
``sorted_x`` go through ``down(silu(x @ W_gate[e]^T) * (x @ W_up[e]^T))``; the
output is unweighted and stays in sorted order; rows past ``offsets[E]`` are
zero.  The reference's three Triton launches and its host-synchronising tile
metadata become: a one-CTA tile-table kernel, the w13 grouped GEMM with the
SwiGLU in its epilogue (``sorted_x`` is read once, the gate/up outputs never
reach HBM), and the w2 grouped GEMM.  ``BLOCK_M/N/K`` are accepted for
signature compatibility; the tile shape is fixed by the tcgen05 kernels
(128 x 256 x 64).
"""

from __future__ import annotations

import torch

from . import ops


def fused_moe_forward(sorted_x: torch.Tensor, offsets: torch.Tensor, W_gate: torch.Tensor,
                      W_up: torch.Tensor, W_down: torch.Tensor, BLOCK_M: int = 64,
                      BLOCK_N: int = 64, BLOCK_K: int = 32) -> torch.Tensor:
    M, H = sorted_x.shape
    E = W_gate.shape[0]
    if offsets.numel() != E + 1:
        raise ValueError(f"offsets must have E+1 = {E + 1} entries")
    off = offsets.to(device=sorted_x.device, dtype=torch.int64).contiguous()
    tiles, num_tiles, mt = ops.tiles_from_offsets(off, M)
    h = ops.grouped_w13_swiglu(sorted_x.contiguous(), tiles, num_tiles, mt, W_gate.contiguous(),
                               W_up.contiguous())
    y = torch.zeros((M, H), dtype=sorted_x.dtype, device=sorted_x.device)
    ops.grouped_w2(h, tiles, num_tiles, mt, W_down.contiguous(), out=y)
    return y


def fused_moe_forward_w4(sorted_x: torch.Tensor, offsets: torch.Tensor, bank) -> torch.Tensor:
    """``fused_moe_forward`` on a 4-bit bank (``W4Experts``): rows
    ``offsets[e]:offsets[e+1]`` of ``sorted_x`` through expert e, unweighted, in
    sorted order; rows before ``offsets[0]`` and from ``offsets[E]`` on are zero."""
    off = offsets.to(device=sorted_x.device, dtype=torch.int64).contiguous()
    return ops.sorted_experts_w4(sorted_x.contiguous(), off, bank)
