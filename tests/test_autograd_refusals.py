"""The operators around the layer are not recorded by autograd: a call whose result would have lost a gradient without a word, or that would write a tensor behind autograd's
back, is refused. (The check comes ahead of all others, so it shows on the CPU, where any call that passes it is refused for its device.)"""
import pytest
import torch

import hopper_megamoe_basedondeepgemm_b200 as mm


def _tensors(device):
    g = torch.Generator().manual_seed(0)

    def randn(*shape):
        return torch.randn(shape, generator=g).to(device)
    return dict(r=randn(6, 64), y=randn(6, 64), w=randn(64), p=randn(64), g=randn(6, 1), o=randn(6, 64), n=randn(6, 64), l=randn(6, 48), k=randn(6, 8), b=randn(48), d=randn(6, 48),
                i=torch.arange(48, device=device).reshape(6, 8))


def _norm(t):
    return mm.block_norm(t['r'], t['y'], pre_weight=t['w'], post_weight=t['p'], gate=t['g'], residual_out=t['o'], normed=t['n'])


def _route(t):
    return mm.route_tokens(t['l'], 8, 1, t['b'], topk_weights=t['k'])


def _balance(t):
    return mm.balance_loss(t['l'], t['i'])


def _gradient(t):
    return mm.router_backward(t['l'], t['i'], d_topk_weights=t['k'], d_logits=t['d'])


CALLS = [(_norm, n) for n in 'rywpgon'] + [(_route, 'l'), (_route, 'k'), (_balance, 'l'), (_gradient, 'd')]


@pytest.mark.parametrize('call, name', CALLS)
def test_tensors_that_require_a_gradient(call, name):
    t = _tensors('cpu')
    t[name].requires_grad_(True)
    with pytest.raises(RuntimeError, match='autograd'):
        call(t)
    t[name] = t[name].detach().requires_grad_(True) * 1.0                  # no leaf, either
    with pytest.raises(RuntimeError, match='autograd'):
        call(t)


@pytest.mark.parametrize('call, name', CALLS + [(_gradient, 'l'), (_gradient, 'k')])
def test_forward_mode(call, name):
    t = _tensors('cpu')
    with torch.autograd.forward_ad.dual_level():
        t[name] = torch.autograd.forward_ad.make_dual(t[name], torch.ones_like(t[name]))
        with pytest.raises(RuntimeError, match='forward-mode'):
            call(t)


@pytest.mark.gpu
def test_calls_that_lose_nothing():
    """Without gradients enabled, on detached tensors, and where only the gradient is asked for."""
    want = {}
    for mode in ('plain', 'no_grad', 'inference', 'detached'):
        t = _tensors('cuda')
        for name in 'rywpglb':
            if mode in ('no_grad', 'inference'):
                t[name].requires_grad_(True)
            elif mode == 'detached':
                t[name] = t[name].requires_grad_(True).detach()
        with torch.inference_mode() if mode == 'inference' else (torch.no_grad() if mode == 'no_grad' else torch.enable_grad()):
            out = [*_norm(t), *_route(t), _balance(t).losses, _gradient(t)]
        assert all(not o.requires_grad for o in out)
        want[mode] = out
    for got in want.values():
        assert all(torch.equal(a, b) for a, b in zip(got, want['plain']))
    t = _tensors('cuda')
    t['b'].requires_grad_(True)                # the choice of experts has no gradient
    assert all(torch.equal(a, b) for a, b in zip(_route(t), want['plain'][2:4]))
    for name in 'rywpg':
        t[name].requires_grad_(True)
    g = mm.block_norm_backward(t['o'], t['n'], t['r'], t['y'], pre_weight=t['w'], post_weight=t['p'], gate=t['g'])
    t['y'].backward(g.y)
    assert torch.equal(t['y'].grad, g.y)
    logits = t['l'].requires_grad_(True) * 1.0  # as a training step by hand has it
    b = mm.balance_loss(logits.detach(), t['i'])
    logits.backward(mm.router_backward(logits, t['i'], balance=b))
    assert bool(t['l'].grad.any())


@pytest.mark.gpu
def test_a_leaf_is_written_only_where_torch_would():
    t = _tensors('cuda')
    t['o'].requires_grad_(True)
    with pytest.raises(RuntimeError, match='autograd'):
        _norm(t)
    with torch.no_grad():
        assert _norm(t)[0] is t['o']
    assert t['o']._version > 0 and t['o'].requires_grad
