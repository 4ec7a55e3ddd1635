"""The residual stream between two blocks: norm, gate and scale of a block's output, sum, and the next block's norm.

A decoder layer of the reference adds its attention's output to the residual
and norms the sum for the MoE block (TF/models/qwen3_moe/modeling_qwen3_moe.py:340-345),
adds the MoE block's output (:347), and the next layer norms that sum again.
``residual_norm`` is one such step: the sum and the norm in one pass over the
rows, with what models put between a block and the residual besides: a norm of
the block's own output, a gate, and scales of either branch.  Where
``norm_router_aux`` starts from a hidden state that is already summed, this
makes both that state and the normed rows that the router and the experts read.
"""

from __future__ import annotations

from torch import Tensor

from . import ops

__all__ = ["residual_norm"]


def residual_norm(
    y: Tensor,
    residual: Tensor,
    weight: Tensor,
    *,
    post_weight: Tensor | None = None,
    gate: Tensor | None = None,
    branch_scale: float = 1.0,
    residual_scale: float = 1.0,
    eps: float = 1e-6,
) -> tuple[Tensor, Tensor]:
    """(hidden, x) for a block's output ``y`` [..., H] and the ``residual`` [..., H] that went around the block:

        hidden = residual_scale * residual + branch_scale * gate * N(y; post_weight)
        x      = N(hidden; weight),     N(v; w) = v * rsqrt(mean(v^2) + eps) * w

    ``post_weight`` [H] norms the block's output (None: y as it is); ``gate`` is
    [..., 1] (a value per token), [H] (per channel), [..., H], or None.  All
    tensors are bfloat16, or all float32; H is a multiple of 8 and at most 8192.
    The arithmetic is fp32 and rounds each output once (x is normed from the
    unrounded sum).  Gradients reach every tensor; the scales and eps are
    numbers, not differentiated."""
    return ops.run_residual_norm(y, residual, weight, post_weight, gate, float(branch_scale), float(residual_scale),
                                 float(eps))
