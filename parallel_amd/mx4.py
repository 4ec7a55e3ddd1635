"""Experts on 4-bit microscaled weights and activations, for inference.

``quantize_mx4`` holds blocks of 32 values as 4-bit floating-point codes with a
shared power-of-two scale (the OCP microscaling format's E2M1 elements with
E8M0 scales): 17 bits for 32 bits of bf16, and the gfx950 matrix cores multiply
such operands directly at four times the bf16 rate.  ``mx4_grouped_mm`` and
``mx4_swiglu`` are the grouped products of the expert path on them, and
``mx4_experts`` / ``MX4Experts`` the whole of it behind the interface that
``Experts`` has (TF/integrations/moe.py:377-478): a layer's experts weigh
17/64 of their bf16 size, which is what a decoding step streams.  The
reference has no 4-bit path; there are no gradients.
"""

from __future__ import annotations

import torch
from torch import Tensor, nn

from . import ops

__all__ = ["MX4Experts", "MX4Tensor", "mx4_experts", "mx4_grouped_mm", "mx4_swiglu", "quantize_mx4"]


class MX4Tensor:
    """A tensor [..., K] of 4-bit microscaled values.

    ``codes`` uint8 [..., K/2] (the value of even index in a byte's low half:
    sign, then the index of 0, 0.5, 1, 1.5, 2, 3, 4, 6) and ``scales`` uint8
    [..., 8 ceil(K/256)], of which byte j stands for 2^(byte - 127) (255: NaN)
    for the values 32 j to 32 j + 31 and the bytes past K/32 pad the row.
    Scales given without padding ([..., K/32], as checkpoints hold them) are
    padded here, once."""

    __slots__ = ("codes", "scales")

    def __init__(self, codes: Tensor, scales: Tensor):
        if not codes.dim() or not scales.dim():
            raise ValueError("MX4Tensor: codes and scales need a dimension of values")
        K = 2 * codes.shape[-1]
        if scales.shape[-1] * 32 == K and scales.shape[-1] != ops.mx4_pitch(K):
            scales = nn.functional.pad(scales, (0, ops.mx4_pitch(K) - scales.shape[-1]))
        ops._check_mx4("MX4Tensor", codes, scales)
        self.codes, self.scales = codes, scales

    @classmethod
    def _of(cls, codes: Tensor, scales: Tensor) -> "MX4Tensor":
        """From parts that an operator made."""
        t = object.__new__(cls)
        t.codes, t.scales = codes, scales
        return t

    @property
    def shape(self) -> torch.Size:
        return self.codes.shape[:-1] + (2 * self.codes.shape[-1],)

    @property
    def device(self) -> torch.device:
        return self.codes.device

    @property
    def block_scales(self) -> Tensor:
        """The scales without padding, [..., K/32]."""
        return self.scales[..., :self.codes.shape[-1] // 16]

    def dequantize(self, dtype: torch.dtype = torch.bfloat16) -> Tensor:
        """The values, exactly, in bfloat16 or float32 (infinity past their range)."""
        if dtype not in (torch.bfloat16, torch.float32):
            raise ValueError(f"4-bit values are given as bfloat16 or float32, not {dtype}")
        return ops.run_mx4("mx4_dequantize", self.codes, self.scales, dtype == torch.float32)

    def to(self, device) -> "MX4Tensor":
        return MX4Tensor(self.codes.to(device), self.scales.to(device))

    def __repr__(self) -> str:
        return f"MX4Tensor({tuple(self.shape)}, device={self.device})"


def quantize_mx4(x: Tensor) -> MX4Tensor:
    """x [..., K] (bfloat16 or float32, K a multiple of 32) in blocks of 32 along the last dimension.

    A block's scale is the power of two that puts its largest size in [4, 8);
    every value is rounded to the nearest code, halfway to the even one, sizes
    past 6 to 6.  A block that holds an infinity or NaN is NaN throughout."""
    return MX4Tensor._of(*ops.run_mx4("mx4_quantize", x))


def mx4_grouped_mm(a: MX4Tensor, w: MX4Tensor, offsets: Tensor) -> Tensor:
    """[M, N] bf16: rows offsets[g-1] .. offsets[g] of a [M, K] times w[g]^T, w [G, N, K] (N a multiple of 8).

    ``offsets`` [G] int32 holds each group's end row (F.grouped_mm's ``offs``).
    Rows from offsets[-1] on are not computed: their values are undefined."""
    return ops.run_mx4("mx4_grouped_mm", a.codes, a.scales, w.codes, w.scales, offsets)


def mx4_swiglu(a: MX4Tensor, w: MX4Tensor, offsets: Tensor) -> Tensor:
    """[M, I] bf16: silu(gate) * up of the same grouped product with w [G, 2I, K], the gate's I rows first."""
    return ops.run_mx4("mx4_grouped_swiglu", a.codes, a.scales, w.codes, w.scales, offsets)


def mx4_experts(hidden: Tensor, top_k_index: Tensor, top_k_weights: Tensor, gate_up: MX4Tensor,
                down: MX4Tensor) -> Tensor:
    """The routed experts [T, H] of hidden [T, H] (bf16 or fp32) on 4-bit weights.

    gate_up [E, 2I, H] and down [E, H, I]; H and I are multiples of 32.  The
    tokens and the act values are quantised too, each rounded once from fp32 or
    the given type; sums are fp32, the experts' rows bf16 as on the bf16 path.
    Ids equal to E (the expert-parallel sentinel) contribute nothing."""
    return ops.run_mx4("mx4_experts", hidden, top_k_index, top_k_weights, gate_up.codes, gate_up.scales, down.codes,
                       down.scales)


class MX4Experts(nn.Module):
    """``Experts`` for inference on 4-bit weights: the same call, the weights as buffers of codes and scales.

    A drop-in for the ``experts`` of ``SparseMoeBlock`` or of a transformers
    block: ``block.experts = MX4Experts.from_experts(block.experts)``.  Call it
    under ``torch.no_grad()``."""

    def __init__(self, gate_up: MX4Tensor, down: MX4Tensor):
        super().__init__()
        self.num_experts, self.hidden_dim, self.intermediate_dim = gate_up.shape[0], gate_up.shape[2], down.shape[2]
        if tuple(gate_up.shape[:2]) != (down.shape[0], 2 * down.shape[2]) or down.shape[1] != self.hidden_dim:
            raise ValueError(f"expert weights do not match: gate_up {tuple(gate_up.shape)}, down {tuple(down.shape)}")
        self.register_buffer("gate_up_codes", gate_up.codes)
        self.register_buffer("gate_up_scales", gate_up.scales)
        self.register_buffer("down_codes", down.codes)
        self.register_buffer("down_scales", down.scales)

    @classmethod
    def from_experts(cls, experts: nn.Module) -> "MX4Experts":
        """Quantises the weights of ``Experts`` or of a transformers experts module (gated SiLU, no biases)."""
        from .moe import _check_gated_silu

        _check_gated_silu(experts)
        with torch.no_grad():
            return cls(quantize_mx4(experts.gate_up_proj), quantize_mx4(experts.down_proj))

    def forward(self, hidden_states: Tensor, top_k_index: Tensor, top_k_weights: Tensor) -> Tensor:
        return ops.run_mx4("mx4_experts", hidden_states, top_k_index, top_k_weights, self.gate_up_codes,
                           self.gate_up_scales, self.down_codes, self.down_scales)
