"""``W4Experts`` — the expert weights of one MoE layer in 4 bits.

Every row of a projection is cut into groups of 32, 64 or 128 columns with a
bf16 scale and, optionally, a zero point each:
``w[n, c] = scale[n, c // group] * (code[n, c] - zero[n, c // group])``, codes
and zero points in 0..15 (zero point 8 throughout where none are kept).  The
bank holds the three projections in the layout the kernels stream
(``moe_w4_pack`` in the C ABI): gate and up interleaved by eight rows, 16-row
tiles of 64-column blocks.  It takes 0.5 byte and the group's share of a scale
per weight, the scales twice, as bf16 and as fp16 multiples of powers of two
(``3 * H * I * (1/2 + 4/group)`` bytes per expert without zero points, and 4 per row).

The kernels multiply activations by 128 + code, or from 8 records per expert on by the
weight in fp16 (rounded by 2^-12 of it at most), and sum in fp32, so K * 144 * |x| has to
stay below 3.4e38; an infinity or a NaN in a row makes the outputs of that row NaN or
infinite and no other's.

Build it once when the weights are loaded, from codes (``from_codes``) or from
bf16 weights (``quantize``); the ops that take it are ``ops.moe_layer_w4``,
``ops.experts_w4``, ``ops.grouped_w13_swiglu_w4``, ``ops.grouped_w2_w4`` and
``fused_moe_forward_w4``.
"""

from __future__ import annotations

import ctypes

import torch

from . import _native, ops

GROUPS = (32, 64, 128)
BLOCK = 64          # columns of a packed block
MAX_COLUMNS = 8192  # of a projection


@torch.no_grad()
def quantize_w4(w: torch.Tensor, group_size: int = 128, symmetric: bool = True):
    """Codes, scales and zero points of ``w`` [..., K] (any float type, any device).

    ``symmetric``: scale = max|w| / 7 of the group, codes round(w / scale) + 8, no
    zero points (the third result is None).  Otherwise the group's range
    (extended to hold 0) is cut into 15 steps and the zero point is the code of 0.
    The scales are rounded to bf16 before the codes are taken, so the codes are
    the nearest to the weights under the scales that are kept."""
    if group_size not in GROUPS:
        raise ValueError(f"group_size must be one of {GROUPS}, got {group_size}")
    K = w.shape[-1]
    if K % group_size:
        raise ValueError(f"the last dimension {K} must be a multiple of the group {group_size}")
    if not w.is_floating_point():
        raise TypeError(f"w must be a floating-point tensor, got {w.dtype}")
    g = w.float().reshape(*w.shape[:-1], K // group_size, group_size)
    if not bool(torch.isfinite(g).all()):
        raise ValueError("w holds an infinity or a NaN")
    if symmetric:
        scales = (g.abs().amax(-1) / 7.0).bfloat16()
        zeros = None
    else:
        lo, hi = g.amin(-1).clamp_max(0.0), g.amax(-1).clamp_min(0.0)
        scales = ((hi - lo) / 15.0).bfloat16()
    s = scales.float()
    if not bool(torch.isfinite(s).all()):
        raise ValueError("a group's range exceeds the scales' type (bfloat16)")
    s = torch.where(s > 0, s, torch.ones_like(s)).unsqueeze(-1)  # a group of zeros: any scale
    if symmetric:
        codes = (g / s).round_().add_(8.0)
    else:
        zeros = (-lo.unsqueeze(-1) / s).round_().clamp_(0, 15)
        codes = (g / s).round_().add_(zeros)
        zeros = zeros.squeeze(-1).to(torch.uint8)
    return codes.clamp_(0, 15).to(torch.uint8).reshape(w.shape), scales, zeros


def dequantize_w4(codes: torch.Tensor, scales: torch.Tensor,
                  zeros: torch.Tensor | None = None) -> torch.Tensor:
    """The fp32 weights that codes, scales and zero points stand for."""
    group = codes.shape[-1] // scales.shape[-1]
    q = codes.float().reshape(*scales.shape, group)
    q = q - (8.0 if zeros is None else zeros.float().unsqueeze(-1))
    return (q * scales.float().unsqueeze(-1)).reshape(codes.shape)


class W4Experts:
    """Packed 4-bit expert weights (w_gate, w_up [E, I, H], w_down [E, H, I])."""

    def __init__(self, w13, w2, num_experts: int, hidden: int, intermediate: int,
                 group_size: int, has_zeros: bool) -> None:
        """Use ``from_codes`` or ``quantize``; w13 and w2 are packed (q, s, f, r), codes and
        scales and the scales again as products of many records read them."""
        self.w13, self.w2 = w13, w2
        self.num_experts, self.hidden, self.intermediate = num_experts, hidden, intermediate
        self.group_size, self.has_zeros = group_size, has_zeros
        self.device = w13[0].device
        fine = [t.data_ptr() for t in (*w13[2:], *w2[2:])]
        self._struct = _native.W4BankStruct(
            *(t.data_ptr() for t in (*w13[:2], *w2[:2])), num_experts, hidden, intermediate,
            group_size, int(has_zeros) | (_native.W4_FINE if fine else 0), *fine)
        self.native = ctypes.addressof(self._struct)  # const moe_w4_bank*

    def __getstate__(self):
        """What a copy or a file holds of a bank: not the addresses of its tensors."""
        return (self.w13, self.w2, self.num_experts, self.hidden, self.intermediate,
                self.group_size, self.has_zeros)

    def __setstate__(self, state) -> None:
        self.__init__(*state)

    def nbytes(self) -> int:
        return sum(t.numel() * t.element_size() for t in (*self.w13, *self.w2))

    @classmethod
    @torch.no_grad()
    def from_codes(cls, w_gate, w_up, w_down, *, into: "W4Experts | None" = None) -> "W4Experts":
        """Each argument is ``(codes, scales, zeros)``: uint8 codes [E, N, K] with one
        code (0..15) per byte, bf16 scales [E, N, K / group], and uint8 zero points
        of the scales' shape or None (for all three projections or for none).
        Synchronises once, to refuse codes or zero points above 15.  ``into``: a bank of
        the same sizes, form and device, whose memory the new one takes over (its values
        change in place, so captured graphs that read it follow); another is not touched."""
        parts = []
        for name, part in (("w_gate", w_gate), ("w_up", w_up), ("w_down", w_down)):
            codes, scales, zeros = part
            ops._need(codes, f"{name} codes", torch.uint8, 3)
            ops._need(scales, f"{name} scales", torch.bfloat16, 3)
            if zeros is not None:
                ops._need(zeros, f"{name} zeros", torch.uint8, 3)
                if zeros.shape != scales.shape:
                    raise ValueError(f"{name}: zero points {tuple(zeros.shape)} must have the "
                                     f"scales' shape {tuple(scales.shape)}")
            parts.append((codes, scales, zeros))
        (gc, gs, gz), (uc, us, uz), (dc, ds, dz) = parts
        E, I, H = gc.shape
        if E == 0 or H == 0 or I == 0:
            raise ValueError("the bank needs at least one expert, row and column")
        if uc.shape != gc.shape or tuple(dc.shape) != (E, H, I):
            raise ValueError(f"codes must be w_gate, w_up [E, I, H] and w_down [E, H, I], got "
                             f"{tuple(gc.shape)}, {tuple(uc.shape)}, {tuple(dc.shape)}")
        if len({gz is None, uz is None, dz is None}) != 1:
            raise ValueError("zero points must come for all three projections or for none")
        group = H // max(gs.shape[2], 1)
        if group not in GROUPS:
            raise ValueError(f"scales {tuple(gs.shape)} of codes {tuple(gc.shape)} give groups of "
                             f"{group} columns; they must be one of {GROUPS}")
        for name, codes, scales in (("w_gate", gc, gs), ("w_up", uc, us), ("w_down", dc, ds)):
            want = (E, codes.shape[1], codes.shape[2] // group)
            if codes.shape[2] % group or tuple(scales.shape) != want:
                raise ValueError(f"{name} scales must be {want} for groups of {group} columns of "
                                 f"codes {tuple(codes.shape)}, got {tuple(scales.shape)}")
        dev = gc.device
        if any(t is not None and t.device != dev for p in parts for t in p):
            raise ValueError("codes, scales and zero points must be on one device")
        with torch.cuda.device(dev):
            status = torch.zeros(1, dtype=torch.int32, device=dev)
            same = into is not None and len(into.w13) == 4 and (E, H, I, group, gz is not None, dev) == (
                into.num_experts, into.hidden, into.intermediate, into.group_size,
                into.has_zeros, into.device)
            w13 = _pack((gc, gs, gz), (uc, us, uz), group, status, into.w13 if same else None)
            w2 = _pack((dc, ds, dz), None, group, status, into.w2 if same else None)
            code = int(status.item())
        if code:
            raise ValueError(f"codes and zero points must be in 0..15 "
                             f"({_native.error_string(code)})")
        return cls(w13, w2, E, H, I, group, gz is not None)

    @classmethod
    @torch.no_grad()
    def quantize(cls, w_gate: torch.Tensor, w_up: torch.Tensor, w_down: torch.Tensor,
                 group_size: int = 128, symmetric: bool = True, *,
                 into: "W4Experts | None" = None) -> "W4Experts":
        """Round stacked bf16 weights (w_gate, w_up [E, I, H], w_down [E, H, I]) to
        4 bits (``quantize_w4``) and pack them, expert by expert.  ``into``: as for
        ``from_codes``."""
        packed = []
        for name, w in (("w_gate", w_gate), ("w_up", w_up), ("w_down", w_down)):
            if not isinstance(w, torch.Tensor) or not w.is_cuda or w.dim() != 3:
                raise ValueError(f"{name} must be a CUDA tensor of three dims")
            rows = [quantize_w4(w[e], group_size, symmetric) for e in range(w.shape[0])]
            codes, scales = (torch.stack([r[i] for r in rows]) for i in (0, 1))
            packed.append((codes, scales, None if symmetric else torch.stack([r[2] for r in rows])))
        return cls.from_codes(*packed, into=into)


def _pack(first, second, group: int, status: torch.Tensor, into=None):
    codes, scales, zeros = first
    E, N, K = codes.shape
    M = N if second is None else 2 * N
    dev = codes.device
    records = E * M * (K // group) * (1 if zeros is None else 2)
    q, s, f, r = into if into is not None else (
        torch.empty(E * M * K // 2, dtype=torch.uint8, device=dev),
        torch.empty(records, dtype=torch.bfloat16, device=dev),
        torch.empty(records, dtype=torch.float16, device=dev),
        torch.empty(E * (M + 1), dtype=torch.float32, device=dev))
    p = ops._p
    c1, s1, z1 = second if second is not None else (None, None, None)
    ops._rc(_native.load().moe_w4_pack(p(codes), p(scales), p(zeros), p(c1), p(s1), p(z1), E, N, K,
                                       group, p(q), p(s), p(status), ops._stream(dev)),
            "moe_w4_pack")
    ops._rc(_native.load().moe_w4_pack_fine(p(scales), p(zeros), p(s1), p(z1), E, N, K, group,
                                            p(f), p(r), ops._stream(dev)), "moe_w4_pack_fine")
    return q, s, f, r


ops._W4Experts = W4Experts
