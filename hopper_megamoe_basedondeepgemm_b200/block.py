"""The norms of a transformer block around the expert-parallel layer, fused with its gate and the residual stream.

Between two blocks a program adds a block's output to the residual stream and normalises the sum for the next one; some models normalise the output
too, gate it (a shared expert's gate per token, a learned scale per channel) or scale it. `block_norm` is all of that in one pass over the rows:
what it leaves in `normed` is what `mega_moe_from_hidden` and `fe_forward` read, and the layer's `y` goes back through it. One token or a prefill
chunk, in place where the program wants it. `block_norm_backward` is its gradient. Neither is recorded by autograd.
"""
import struct
from typing import NamedTuple, Optional, Tuple

import torch

from . import _lib

MAX_HIDDEN = 8192
_DTYPE = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
_NORM_ARGS = struct.Struct('@7P6q6i3f0P')         # mm_block_norm_args_t
_GRAD_ARGS = struct.Struct('@7P5qPq')             # mm_block_norm_grads_t


def call(device: int, entry: str, *args) -> None:
    """The library's `entry` with `args` and the current stream of `device`, which is the current device while it runs."""
    fn = getattr(_lib.load(), entry)
    if device == torch._C._cuda_getDevice():
        status = fn(*args, torch._C._cuda_getCurrentRawStream(device))
    else:
        with torch.cuda.device(device):
            status = fn(*args, torch._C._cuda_getCurrentRawStream(device))
    if status:
        _lib.check(status, entry[3:])


def _rows(t: torch.Tensor, name: str, shape, dtype, device: int):
    """Address and row stride of a [tokens, hidden] tensor whose rows are packed."""
    if t.shape != shape or t.dtype != dtype:
        raise RuntimeError(f'{name} must be {dtype} {list(shape)}')
    if t.get_device() != device:
        raise RuntimeError(f'{name} must be on the GPU of the other tensors')
    stride, inner = t.stride()
    if inner != 1 and shape[1] > 1:
        raise RuntimeError(f'the channels of {name} must lie next to each other')
    return t.data_ptr(), stride


def _weight(t: Optional[torch.Tensor], name: str, hidden: int, dtype, device: int) -> int:
    if t is None:
        return 0
    if t.shape != (hidden,) or (t.dtype != dtype and t.dtype != torch.float32) or t.get_device() != device or not t.is_contiguous():
        raise RuntimeError(f'{name} must be a contiguous [hidden] tensor of the type of the activations or fp32, on their GPU')
    return t.data_ptr()


def _gate(gate: Optional[torch.Tensor], tokens: int, hidden: int, dtype, device: int):
    """(address, row stride, mode) of a gate: [hidden] per channel, [tokens, 1] per token, [tokens, hidden] per element."""
    if gate is None:
        return 0, 0, 0
    shape = gate.shape
    if (gate.dtype != dtype and gate.dtype != torch.float32) or gate.get_device() != device:
        raise RuntimeError('gate must be of the type of the activations or fp32, on their GPU')
    if len(shape) == 1 and shape[0] == hidden and gate.is_contiguous():
        return gate.data_ptr(), 0, 1
    if len(shape) == 2 and shape[0] == tokens:
        if shape[1] == hidden and (hidden == 1 or gate.stride(1) == 1):
            return gate.data_ptr(), gate.stride(0), 3
        if shape[1] == 1:
            return gate.data_ptr(), gate.stride(0), 2
    raise RuntimeError('gate must be [hidden], [tokens, 1] or [tokens, hidden], its channels next to each other')


def _block(residual, y, pre_weight, post_weight, gate, dtype):
    """What both directions check: (tokens, hidden, device, and the addresses, strides and types of the inputs)."""
    if residual.dim() != 2 or not residual.is_cuda or residual.dtype not in _DTYPE or dtype not in _DTYPE:
        raise RuntimeError('residual must be a CUDA [tokens, hidden] tensor; types are bf16, fp16 and fp32')
    if residual.dtype != dtype and residual.dtype != torch.float32:
        raise RuntimeError('the residual stream must be of the type of the activations or fp32')
    shape = residual.shape
    tokens, hidden = shape
    if hidden < 1 or hidden > MAX_HIDDEN:
        raise RuntimeError(f'hidden must be 1 to {MAX_HIDDEN}')
    if y is None and (gate is not None or post_weight is not None or pre_weight is None):
        raise RuntimeError('without y there is only the norm of the stream: pre_weight, and neither post_weight nor gate')
    if pre_weight is not None and post_weight is not None and pre_weight.dtype != post_weight.dtype:
        raise RuntimeError('both weights must be of one type')
    device = residual.get_device()
    r_ptr, r_ld = _rows(residual, 'residual', shape, residual.dtype, device)
    y_ptr, y_ld = _rows(y, 'y', shape, dtype, device) if y is not None else (0, 0)
    pre, post = _weight(pre_weight, 'pre_weight', hidden, dtype, device), _weight(post_weight, 'post_weight', hidden, dtype, device)
    g_ptr, g_ld, g_mode = _gate(gate, tokens, hidden, dtype, device)
    x = _DTYPE[dtype]
    w = pre_weight if pre_weight is not None else post_weight
    types = (x, _DTYPE[residual.dtype], x if w is None else _DTYPE[w.dtype], x if gate is None else _DTYPE[gate.dtype], g_mode)
    return shape, device, (r_ptr, y_ptr, g_ptr, pre, post), (r_ld, y_ld, g_ld), types


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
    that of the given `normed`, or of the stream). Sums of squares are kept in 32 bits, which hold values up to about 1e17.
    """
    dtype = y.dtype if y is not None else (normed.dtype if normed is not None else residual.dtype)
    shape, device, ptrs, lds, types = _block(residual, y, pre_weight, post_weight, gate, dtype)
    out_ptr = out_ld = normed_ptr = normed_ld = 0
    if y is not None:
        if residual_out is None:
            residual_out = torch.empty_like(residual)
        out_ptr, out_ld = _rows(residual_out, 'residual_out', shape, residual.dtype, device)
    elif residual_out is not None:
        raise RuntimeError('without y the stream stays as it is: no residual_out')
    if pre_weight is not None:
        if normed is None:
            normed = torch.empty_like(residual) if y is None else torch.empty_like(y)
        normed_ptr, normed_ld = _rows(normed, 'normed', shape, dtype, device)
    elif normed is not None:
        raise RuntimeError('normed needs pre_weight')
    call(device, 'mm_block_norm', _NORM_ARGS.pack(*ptrs, out_ptr, normed_ptr, shape[0], *lds, out_ld, normed_ld, shape[1], *types, scale, eps, weight_offset))
    return (residual if y is None else residual_out), normed


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
    if (d_normed is None) != (pre_weight is None):
        raise RuntimeError('d_normed goes with pre_weight')
    if d_normed is None and d_residual_out is None:
        raise RuntimeError('the gradient of at least one output must be given')
    dtype = y.dtype if y is not None else (d_normed.dtype if d_normed is not None else residual.dtype)
    shape, device, ptrs, lds, types = _block(residual, y, pre_weight, post_weight, gate, dtype)
    tokens, hidden = shape
    dro_ptr, dro_ld = _rows(d_residual_out, 'd_residual_out', shape, residual.dtype, device) if d_residual_out is not None else (0, 0)
    dn_ptr, dn_ld = _rows(d_normed, 'd_normed', shape, dtype, device) if d_normed is not None else (0, 0)
    d_residual = torch.empty_like(residual)
    d_y = torch.empty_like(y) if y is not None else None
    d_gate = torch.empty_like(gate) if gate is not None else None
    d_pre = torch.empty_like(pre_weight) if pre_weight is not None else None
    d_post = torch.empty_like(post_weight) if post_weight is not None else None
    ws_ptr = ws_bytes = 0
    if tokens and (d_pre is not None or d_post is not None or types[4] == 1):
        ws_bytes = _lib.load().mm_block_norm_workspace_bytes(tokens, hidden)
        workspace = residual.new_empty(ws_bytes, dtype=torch.uint8)
        ws_ptr = workspace.data_ptr()
    args = _NORM_ARGS.pack(*ptrs, 0, 0, tokens, *lds, 0, 0, hidden, *types, scale, eps, weight_offset)
    grads = _GRAD_ARGS.pack(dro_ptr, dn_ptr, d_residual.data_ptr(), d_y.data_ptr() if d_y is not None else 0, d_gate.data_ptr() if d_gate is not None else 0,
                            d_pre.data_ptr() if d_pre is not None else 0, d_post.data_ptr() if d_post is not None else 0,
                            dro_ld, dn_ld, hidden, hidden, 1 if types[4] == 2 else hidden, ws_ptr, ws_bytes)
    call(device, 'mm_block_norm_backward', args, grads)
    return BlockNormGrads(d_residual, d_y, d_gate, d_pre, d_post)
