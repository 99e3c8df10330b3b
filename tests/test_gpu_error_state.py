"""A call that fails leaves the ones after it alone: what CUDA said to the first is not taken for the result of a launch that went well."""
import ctypes

import pytest
import torch

import hopper_megamoe_basedondeepgemm_b200 as mm
from hopper_megamoe_basedondeepgemm_b200 import _lib, quant

pytestmark = pytest.mark.gpu


def _fail():
    """A window larger than any GPU: refused by CUDA's allocator, without harm."""
    lib, p, handle = _lib.load(), ctypes.c_void_p(), ctypes.create_string_buffer(64)
    assert lib.mm_window_alloc(1 << 55, ctypes.byref(p), handle) == 3
    assert b'out of memory' in lib.mm_last_cuda_error()


def _cast(x):
    packed, sf = torch.empty((x.shape[0], x.shape[1] // 2), dtype=torch.uint8, device='cuda'), torch.empty((x.shape[0], x.shape[1] // 32), device='cuda')
    _lib.check(_lib.load().mm_cast_rows_to_fp4(x.data_ptr(), 0, x.shape[0], x.shape[1], 32, 1, packed.data_ptr(), sf.data_ptr(), None), 'mm_cast_rows_to_fp4')
    return packed


@pytest.mark.parametrize('call', ['route', 'balance', 'balance of many', 'balance of very many', 'gradient', 'norm', 'norm gradient', 'cast', 'absmax', 'weights'])
def test_calls_behind_a_failed_one(call):
    logits = torch.randn((500, 384), device='cuda')
    idx, _ = mm.route_tokens(logits, 8)
    b = mm.balance_loss(logits, idx)
    x, w = torch.randn((40, 256), device='cuda'), torch.ones(256, device='cuda')
    weights = quant.cast_grouped_weights_to_fp4(torch.randn((2, 256, 256), device='cuda').bfloat16(), 'mxfp4')
    cu = torch.arange(0, 501, 10, dtype=torch.int32, device='cuda')
    calls = {'route': lambda: mm.route_tokens(logits, 8)[0], 'balance': lambda: mm.balance_loss(logits[:20], idx[:20]).counts, 'balance of many': lambda: mm.balance_loss(logits, idx).counts,
             'balance of very many': lambda: mm.balance_loss(logits, idx, cu_seqlens=cu).counts, 'gradient': lambda: mm.router_backward(logits, idx, balance=b),
             'norm': lambda: mm.block_norm(x, x, pre_weight=w)[1], 'norm gradient': lambda: mm.block_norm_backward(x, x, x, x, pre_weight=w).pre_weight,
             'cast': lambda: _cast(x), 'absmax': lambda: mm.nvfp4_global_scale(x),
             'weights': lambda: mm.transform_weights_for_mega_moe(weights, weights)[0][0]}
    f = calls[call]
    want = f()
    _fail()
    got = f()
    torch.cuda.synchronize()
    assert torch.equal(got, want) if isinstance(got, torch.Tensor) else got == want
