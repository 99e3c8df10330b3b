"""Routing from logits, the balance loss over the experts, and the gradient of both.

`fe_forward` and `mega_moe_from_hidden` route from bf16 hidden states inside the library. A program that has logits of its own (a 32-bit router, noise
on the scores, experts that are switched off, padding) gets the same top-k and weights from `route_tokens`, into the buffer's views if it likes;
in training `balance_loss` adds up how the experts are used, and `router_backward` is the logits' gradient of both in one pass. Nothing here is
recorded by autograd: `route_tokens` and `balance_loss` refuse logits that require a gradient while gradients are enabled (a training step calls them from a
`torch.autograd.Function`, or on detached logits, and hands what `router_backward` returns to `logits.backward`). `router_backward` takes such logits; its result has no
further derivative.
"""
from typing import Optional, Tuple, Union

import torch

from ._binding import binding


def route_tokens(logits: torch.Tensor, topk: int, score_mode: int = 0, expert_bias: Optional[torch.Tensor] = None, *, valid: Optional[torch.Tensor] = None,
                 route_scale: float = 1.0, topk_idx: Optional[torch.Tensor] = None,
                 topk_weights: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """`(topk_idx int64, topk_weights fp32)`, both `[tokens, topk]`, of bf16, fp16 or fp32 logits `[tokens, experts]`.

    score_mode 0: the largest logits; weights are the softmax over the selected ones. 1: the largest `sigmoid(logit) + expert_bias` (fp32
    `[experts]`, optional), compared as in 64 bits; weights are the sigmoids over their sum, also where these are smaller than 32 bits hold (and 0 where they are 0 in
    64: all selected logits below -709). Both times `route_scale`. Experts come in descending order, equal ones lower index first. A logit of -inf or NaN switches an expert off for the token, a bias of -inf or NaN for all. Slots for which no expert is left,
    and tokens whose `valid` (bool or uint8 `[tokens]`) is 0, get index -1 and weight 0: the layer's masked slots. `topk_idx` / `topk_weights` may
    be given, e.g. `sym_buffer.topk_idx[:tokens]`, apart from everything that the call reads. At most 1024 experts and 32 routes per token.
    """
    return binding.route_tokens(logits, topk, score_mode, expert_bias, valid, route_scale, topk_idx, topk_weights)


class BalanceLoss:
    """What `balance_loss` returns, and `router_backward` takes.

    losses      fp32 [3]: balance_coef * balance + z_coef * z, balance, z (no graph: `router_backward` has their gradient)
    counts      int32 [sequences, experts]: routing slots per expert
    mean_probs  fp32 [sequences, experts]: mean probability of the expert over the sequence's routed tokens (summed in steps of 2^-63 of the next power of two above the number
                of tokens)
    tokens      int32 [sequences]: tokens with a route
    """
    __slots__ = ('losses', 'counts', 'mean_probs', 'tokens', 'cu_seqlens', 'balance_coef', 'z_coef', 'score_mode')

    def __init__(self, losses, counts, mean_probs, tokens, cu_seqlens, balance_coef, z_coef, score_mode):
        self.losses, self.counts, self.mean_probs, self.tokens = losses, counts, mean_probs, tokens
        self.cu_seqlens, self.balance_coef, self.z_coef, self.score_mode = cu_seqlens, balance_coef, z_coef, score_mode

    @property
    def loss(self) -> torch.Tensor:
        return self.losses[0]


def balance_loss(logits: torch.Tensor, topk_idx: torch.Tensor, score_mode: int = 0, *, cu_seqlens: Optional[torch.Tensor] = None,
                 balance_coef: float = 1.0, z_coef: float = 0.0) -> BalanceLoss:
    """Balance loss of a router over its experts, with per-expert counts.

    A token's probabilities p are the softmax of its logits (score_mode 0) or their sigmoids over their sum (1), over all experts. With c_e the slots
    of `topk_idx` (int64 `[tokens, topk]`) that name expert e, n the tokens with at least one such slot, and P_e the mean of p_e over them,

        balance = sum_e (experts * c_e / (topk * n)) * P_e          z = mean of log(sum exp logits)^2 over the n tokens

    `losses[0] = balance_coef * balance + z_coef * z`. With `cu_seqlens` (int32 `[sequences + 1]`, ascending) counts, n and P are those of each
    sequence and `balance` is the mean over the sequences that have such tokens; tokens outside of all sequences count nowhere. Slots outside of
    0..experts-1 (masked ones) are no routes; an expert that a token names twice counts twice. The results are the same in every call.
    """
    return BalanceLoss(*binding.balance_loss(logits, topk_idx, score_mode, cu_seqlens, balance_coef, z_coef), cu_seqlens, balance_coef, z_coef, score_mode)


def router_backward(logits: torch.Tensor, topk_idx: torch.Tensor, score_mode: int = 0, *, d_topk_weights: Optional[torch.Tensor] = None,
                    route_scale: float = 1.0, balance: Optional[BalanceLoss] = None, d_loss: Union[float, torch.Tensor] = 1.0,
                    d_logits: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Gradient of `sum(d_topk_weights * topk_weights) + d_loss * balance.loss` with respect to the logits, in one pass over them.

    `d_topk_weights` (fp32 `[tokens, topk]`) belongs to the weights of `route_tokens` for `topk_idx` and `route_scale`; the choice of experts, and the
    bias that takes part in it, have no gradient. `balance` is what `balance_loss` returned for the same logits and indices. Either may be left
    out. `d_loss` is a number, or an fp32 tensor with one element on the GPU. Where the tokens of a batch lie on several ranks and it is balanced as a whole,
    `balance.counts` and `balance.tokens` may be summed over the ranks in between: the result is then the gradient of the loss over all of them.
    `d_logits` (the logits' type and shape) may be given, and may be `logits`, but nothing else that the call reads.
    """
    if balance is None:
        return binding.router_backward(logits, topk_idx, score_mode, d_topk_weights, route_scale, None, None, None, 0.0, 0.0, d_loss, d_logits)
    if balance.score_mode != score_mode:
        raise RuntimeError('balance must come from balance_loss with the same score_mode')
    return binding.router_backward(logits, topk_idx, score_mode, d_topk_weights, route_scale, balance.counts, balance.tokens, balance.cu_seqlens,
                                   balance.balance_coef, balance.z_coef, d_loss, d_logits)
