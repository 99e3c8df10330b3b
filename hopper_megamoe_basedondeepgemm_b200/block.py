"""The norms of a transformer block around the expert-parallel layer, fused with its gate and the residual stream.

Between two blocks a program adds a block's output to the residual stream and normalises the sum for the next one; some models normalise the output
too, gate it (a shared expert's gate per token, a learned scale per channel) or scale it. `block_norm` is all of that in one pass over the rows:
what it leaves in `normed` is what `mega_moe_from_hidden` and `fe_forward` read, and the layer's `y` goes back through it. One token or a prefill
chunk, in place where the program wants it. `block_norm_backward` is its gradient. Neither is recorded by autograd: `block_norm` refuses tensors that require a gradient while
gradients are enabled (a training step calls the pair from a `torch.autograd.Function`, or on detached tensors). `block_norm_backward` takes them; its results have no
further derivative.
"""
from typing import NamedTuple, Optional, Tuple

import torch

from ._binding import binding


def block_norm(residual: torch.Tensor, y: Optional[torch.Tensor] = None, *, pre_weight: Optional[torch.Tensor] = None,
               post_weight: Optional[torch.Tensor] = None, gate: Optional[torch.Tensor] = None, scale: float = 1.0, eps: float = 1e-6,
               weight_offset: float = 0.0, residual_out: Optional[torch.Tensor] = None,
               normed: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """`(residual_out, normed)` of `[tokens, hidden]` rows:

        u            = y,  or  y * rsqrt(mean(y^2) + eps) * (weight_offset + post_weight)
        residual_out = residual + scale * gate * u
        normed       = residual_out * rsqrt(mean(residual_out^2) + eps) * (weight_offset + pre_weight)

    in 32 bits, each output rounded once (`normed` is of the sum before it is rounded). bf16, fp16 or fp32 activations; the stream, the weights and
    the gate are of that type or fp32. `gate`: `[hidden]`, `[tokens, 1]`, `[tokens, hidden]` or none. Rows may be strided; hidden is at most 8192.
    Without `y` the stream is only normalised, and returned as it is; without `pre_weight` there is no `normed` (None). `residual_out` may be
    `residual` and `normed` may be `y` or `residual` (the same rows); any other overlap is refused. `normed` has the type of `y` (without `y`:
    that of the given `normed`, or of the stream). Sums of squares are kept in 32 bits, which hold values up to about 1e17;
    `eps` is at least 2^-126, so that squares too small for 32 bits vanish beside it.
    """
    return binding.block_norm(residual, y, pre_weight, post_weight, gate, scale, eps, weight_offset, residual_out, normed)


class BlockNormGrads(NamedTuple):
    """Gradients of `block_norm`, each of the type and shape of what it belongs to; None for what the call did not have."""
    residual: torch.Tensor
    y: Optional[torch.Tensor]
    gate: Optional[torch.Tensor]
    pre_weight: Optional[torch.Tensor]
    post_weight: Optional[torch.Tensor]


def block_norm_backward(d_residual_out: Optional[torch.Tensor], d_normed: Optional[torch.Tensor], residual: torch.Tensor, y: Optional[torch.Tensor] = None,
                        *, pre_weight: Optional[torch.Tensor] = None, post_weight: Optional[torch.Tensor] = None, gate: Optional[torch.Tensor] = None,
                        scale: float = 1.0, eps: float = 1e-6, weight_offset: float = 0.0) -> BlockNormGrads:
    """Gradients of `block_norm` with the same inputs, from those of its outputs: `d_residual_out` (None: zero; without `y`, what the stream gets from
    elsewhere) and `d_normed` (given exactly if `pre_weight` is). Nothing needs to be kept of the forward call but its inputs. Sums over the tokens
    are kept in 32 bits and added in the same order in every call."""
    return BlockNormGrads(*binding.block_norm_backward(d_residual_out, d_normed, residual, y, pre_weight, post_weight, gate, scale, eps, weight_offset))
