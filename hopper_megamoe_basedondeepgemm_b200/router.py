"""Routing from logits, the balance loss over the experts, and the gradient of both.

`fe_forward` and `mega_moe_from_hidden` route from bf16 hidden states inside the library. A program that has logits of its own (a 32-bit router, noise
on the scores, experts that are switched off, padding) gets the same top-k and weights from `route_tokens`, into the buffer's views if it likes;
in training `balance_loss` adds up how the experts are used, and `router_backward` is the logits' gradient of both in one pass. Nothing here is
recorded by autograd.
"""
import struct
from typing import Optional, Tuple, Union

import torch

from . import _lib
from .block import _DTYPE, call

MAX_EXPERTS, MAX_TOPK = 1024, 32
_ROUTER_ARGS = struct.Struct('@3Pq5if')           # mm_router_args_t
_BALANCE_ARGS = struct.Struct('@Piff4P')          # mm_balance_args_t


def _logits(logits: torch.Tensor, topk: int, score_mode: int):
    """(tokens, experts, device, row stride) of the logits, checked with what every call says about them."""
    if logits.dim() != 2 or not logits.is_cuda or logits.dtype not in _DTYPE:
        raise RuntimeError('logits must be a CUDA bf16, fp16 or fp32 [tokens, experts] tensor')
    tokens, experts = logits.shape
    stride, inner = logits.stride()
    if (inner != 1 and experts > 1) or (stride < experts and tokens > 1):
        raise RuntimeError('the logits of a token must lie next to each other, and apart from other tokens\'')
    if not 1 <= topk <= min(experts, MAX_TOPK) or experts > MAX_EXPERTS:
        raise RuntimeError(f'topk must be 1 to {MAX_TOPK} of at most {MAX_EXPERTS} experts')
    if score_mode != 0 and score_mode != 1:
        raise RuntimeError('score_mode must be 0 (softmax) or 1 (sigmoid)')
    return tokens, experts, logits.get_device(), stride


def _plain(t: torch.Tensor, name: str, shape, dtype, device: int) -> int:
    if t.shape != shape or t.dtype != dtype or t.get_device() != device or not t.is_contiguous():
        raise RuntimeError(f'{name} must be a contiguous {dtype} {list(shape)} tensor on the GPU of the logits')
    return t.data_ptr()


def route_tokens(logits: torch.Tensor, topk: int, score_mode: int = 0, expert_bias: Optional[torch.Tensor] = None, *, valid: Optional[torch.Tensor] = None,
                 route_scale: float = 1.0, topk_idx: Optional[torch.Tensor] = None,
                 topk_weights: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """`(topk_idx int64, topk_weights fp32)`, both `[tokens, topk]`, of bf16, fp16 or fp32 logits `[tokens, experts]`.

    score_mode 0: the largest logits; weights are the softmax over the selected ones. 1: the largest `sigmoid(logit) + expert_bias` (fp32
    `[experts]`, optional), compared as in 64 bits; weights are the sigmoids over their sum. Both times `route_scale`. Experts come in descending
    order, equal ones lower index first. A logit of -inf or NaN switches an expert off for the token. Slots for which no expert is left, and
    tokens whose `valid` (bool or uint8 `[tokens]`) is 0, get index -1 and weight 0: the layer's masked slots. `topk_idx` / `topk_weights` may
    be given, e.g. `sym_buffer.topk_idx[:tokens]`. At most 1024 experts and 32 routes per token.
    """
    tokens, experts, device, stride = _logits(logits, topk, score_mode)
    if expert_bias is not None and score_mode != 1:
        raise RuntimeError('expert_bias goes with score_mode 1')
    bias = _plain(expert_bias, 'expert_bias', (experts,), torch.float32, device) if expert_bias is not None else None
    mask = None
    if valid is not None:
        mask = _plain(valid, 'valid', (tokens,), torch.uint8 if valid.dtype == torch.uint8 else torch.bool, device)
    shape = (tokens, topk)
    if topk_idx is None:
        topk_idx = torch.empty(shape, dtype=torch.int64, device=logits.device)
    if topk_weights is None:
        topk_weights = torch.empty(shape, dtype=torch.float32, device=logits.device)
    args = _ROUTER_ARGS.pack(logits.data_ptr(), _plain(topk_idx, 'topk_idx', shape, torch.int64, device),
                             _plain(topk_weights, 'topk_weights', shape, torch.float32, device), stride, tokens, experts, topk, _DTYPE[logits.dtype],
                             score_mode, route_scale)
    call(device, 'mm_route_tokens', args, bias, mask)
    return topk_idx, topk_weights


class BalanceLoss:
    """What `balance_loss` returns, and `router_backward` takes.

    losses      fp32 [3]: balance_coef * balance + z_coef * z, balance, z
    counts      int32 [sequences, experts]: routing slots per expert
    mean_probs  fp32 [sequences, experts]: mean probability of the expert over the sequence's routed tokens
    tokens      int32 [sequences]: tokens with a route
    """
    __slots__ = ('losses', 'counts', 'mean_probs', 'tokens', 'cu_seqlens', 'balance_coef', 'z_coef', 'score_mode')

    def __init__(self, losses, counts, mean_probs, tokens, cu_seqlens, balance_coef, z_coef, score_mode):
        self.losses, self.counts, self.mean_probs, self.tokens = losses, counts, mean_probs, tokens
        self.cu_seqlens, self.balance_coef, self.z_coef, self.score_mode = cu_seqlens, balance_coef, z_coef, score_mode

    @property
    def loss(self) -> torch.Tensor:
        return self.losses[0]

    def _pack(self) -> bytes:
        return _BALANCE_ARGS.pack(0 if self.cu_seqlens is None else self.cu_seqlens.data_ptr(), self.counts.shape[0], self.balance_coef, self.z_coef,
                                  self.counts.data_ptr(), self.tokens.data_ptr(), self.mean_probs.data_ptr(), self.losses.data_ptr())


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
    if topk_idx.dim() != 2:
        raise RuntimeError('topk_idx must be [tokens, topk]')
    topk = topk_idx.shape[1]
    tokens, experts, device, stride = _logits(logits, topk, score_mode)
    idx = _plain(topk_idx, 'topk_idx', (tokens, topk), torch.int64, device)
    sequences = 1
    if cu_seqlens is not None:
        if cu_seqlens.dim() != 1 or cu_seqlens.shape[0] < 2:
            raise RuntimeError('cu_seqlens must be int32 [sequences + 1]')
        _plain(cu_seqlens, 'cu_seqlens', cu_seqlens.shape, torch.int32, device)
        sequences = cu_seqlens.shape[0] - 1
    dev = logits.device
    b = BalanceLoss(torch.empty(3, dtype=torch.float32, device=dev), torch.empty((sequences, experts), dtype=torch.int32, device=dev),
                    torch.empty((sequences, experts), dtype=torch.float32, device=dev), torch.empty(sequences, dtype=torch.int32, device=dev),
                    cu_seqlens, balance_coef, z_coef, score_mode)
    nbytes = _lib.load().mm_balance_workspace_bytes(experts, sequences)
    workspace = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    args = _ROUTER_ARGS.pack(logits.data_ptr(), idx, 0, stride, tokens, experts, topk, _DTYPE[logits.dtype], score_mode, 1.0)
    call(device, 'mm_balance_loss', args, b._pack(), workspace.data_ptr(), nbytes)
    return b


def router_backward(logits: torch.Tensor, topk_idx: torch.Tensor, score_mode: int = 0, *, d_topk_weights: Optional[torch.Tensor] = None,
                    route_scale: float = 1.0, balance: Optional[BalanceLoss] = None, d_loss: Union[float, torch.Tensor] = 1.0,
                    d_logits: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Gradient of `sum(d_topk_weights * topk_weights) + d_loss * balance.loss` with respect to the logits, in one pass over them.

    `d_topk_weights` (fp32 `[tokens, topk]`) belongs to the weights of `route_tokens` for `topk_idx` and `route_scale`; the choice of experts, and the
    bias that takes part in it, have no gradient. `balance` is what `balance_loss` returned for the same logits and indices. Either may be left
    out. `d_loss` is a number, or an fp32 tensor with one element on the GPU. Where the tokens of a batch lie on several ranks and it is balanced as a whole,
    `balance.counts` and `balance.tokens` may be summed over the ranks in between: the result is then the gradient of the loss over all of them.
    `d_logits` (the logits' type and shape) may be given, and may be `logits`.
    """
    if d_topk_weights is None and balance is None:
        raise RuntimeError('d_topk_weights or balance must be given')
    if topk_idx.dim() != 2:
        raise RuntimeError('topk_idx must be [tokens, topk]')
    topk = topk_idx.shape[1]
    tokens, experts, device, stride = _logits(logits, topk, score_mode)
    shape = (tokens, topk)
    idx = _plain(topk_idx, 'topk_idx', shape, torch.int64, device)
    dw = _plain(d_topk_weights, 'd_topk_weights', shape, torch.float32, device) if d_topk_weights is not None else None
    packed = d_loss_ptr = None
    if balance is not None:
        if balance.score_mode != score_mode or balance.counts.shape[1] != experts or balance.counts.get_device() != device:
            raise RuntimeError('balance must come from balance_loss with the same experts and score_mode, on the GPU of the logits')
        packed = balance._pack()
    if isinstance(d_loss, torch.Tensor):
        if d_loss.numel() != 1 or d_loss.dtype != torch.float32 or d_loss.get_device() != device:
            raise RuntimeError('d_loss must be a number or an fp32 tensor with one element on the GPU of the logits')
        d_loss_ptr, d_loss = d_loss.data_ptr(), 0.0
    if d_logits is None:
        d_logits = torch.empty((tokens, experts), dtype=logits.dtype, device=logits.device)
    elif d_logits.shape != logits.shape or d_logits.dtype != logits.dtype or d_logits.get_device() != device or (experts > 1 and d_logits.stride(1) != 1):
        raise RuntimeError('d_logits must be like the logits')
    args = _ROUTER_ARGS.pack(logits.data_ptr(), idx, 0, stride, tokens, experts, topk, _DTYPE[logits.dtype], score_mode, route_scale)
    call(device, 'mm_router_backward', args, dw, packed, d_loss, d_loss_ptr, d_logits.data_ptr(), d_logits.stride(0))
    return d_logits
