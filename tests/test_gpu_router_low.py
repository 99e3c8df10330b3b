"""Sigmoid scores of tokens whose logits are all far below zero: the weights, probabilities and gradients are those of scores over their sum, although the
scores by themselves are below what 32 bits hold (plain forms and tolerances: test_gpu_router, util_block)."""
import pytest
import torch

import hopper_megamoe_basedondeepgemm_b200 as mm
from tests.test_gpu_router import BF16, FP16, FP32, _bias, _check_balance, _check_gradient, _check_route, _logits

pytestmark = pytest.mark.gpu

OFFSETS = [-10.0, -16.0, -17.5, -20.0, -39.0, -41.0, -60.0, -80.0, -87.0, -88.0, -90.0, -104.0, -200.0, -690.0]


def _low(repeat, experts, dtype):
    """Tokens around each offset, `repeat` times."""
    offsets = torch.tensor(OFFSETS, device='cuda').repeat(repeat)[:, None]
    return (_logits(len(offsets), experts, seed=experts) + offsets).to(dtype)


@pytest.mark.parametrize('experts, topk', [(8, 8), (48, 8), (96, 8), (384, 8), (600, 20)])
@pytest.mark.parametrize('dtype', [FP32, BF16, FP16])
@pytest.mark.parametrize('repeat', [1, 40])
def test_low_logits(experts, topk, dtype, repeat):
    logits = _low(repeat, experts, dtype)
    for bias in (None, _bias(experts)):
        out = mm.route_tokens(logits, topk, 1, bias, route_scale=2.5)
        _check_route(logits, topk, 1, bias, None, 2.5, out)
        assert bool((out[1].sum(dim=1) - 2.5).abs().max() <= 2.5 * (topk + 32) * 2.0 ** -24)
    idx = out[0]
    cu = torch.tensor([0, 3, len(logits) // 2, len(logits)], dtype=torch.int32, device='cuda')
    dw = _logits(len(logits), topk, seed=4)
    for ends in (None, cu):
        b = mm.balance_loss(logits, idx, 1, cu_seqlens=ends, balance_coef=0.3, z_coef=0.02)
        _check_balance(logits, idx, 1, ends, 0.3, 0.02, b)
        assert bool((b.mean_probs.sum(dim=1) - 1.0).abs().max() <= (experts + 256) * 2.0 ** -24)
        d = mm.router_backward(logits, idx, 1, d_topk_weights=dw, route_scale=2.5, balance=b, d_loss=1.7)
        _check_gradient(logits, idx, 1, ends, 0.3, 0.02, 2.5, dw, 1.7, d)
    _check_gradient(logits, idx, 1, None, None, None, 1.5, dw, None, mm.router_backward(logits, idx, 1, d_topk_weights=dw, route_scale=1.5))


def test_below_64_bits():
    """Scores that are 0 in 64 bits, too, are 0: no weights, no probabilities, no gradient; experts that are off beside low ones stay off."""
    logits = _logits(6, 48) - 800.0
    logits[1] = torch.finfo(FP32).min
    logits[2:4] += 700.0
    logits[2, 8:] = -float('inf')
    logits[3, ::2] = float('nan')
    idx, w = mm.route_tokens(logits, 8, 1)
    assert bool((idx >= 0).all()) and not w[[0, 1, 4, 5]].any()
    assert bool((w[2:4].sum(dim=1) - 1.0).abs().max() <= 40 * 2.0 ** -24)
    b = mm.balance_loss(logits, idx, 1)
    assert bool((b.mean_probs.sum() - 2.0 / 6.0).abs() <= 300 * 2.0 ** -24) and b.tokens.tolist() == [6]
    d = mm.router_backward(logits, idx, 1, d_topk_weights=_logits(6, 8, seed=3), balance=b)
    assert not d[[0, 1, 4, 5]].any() and d.isfinite().all() and bool(d[2, :8].any()) and not d[2, 8:].any() and not d[3, ::2].any()
