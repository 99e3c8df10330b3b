"""`block_norm` and its gradient over the range of magnitudes that they take: streams of up to 10^17, rows of zeros and of tiny numbers under a small eps. Without a gradient
of the stream from elsewhere, which would be far larger than what the norm gives and hide it (plain form and tolerances: util_block)."""
import pytest
import torch

import hopper_megamoe_basedondeepgemm_b200 as mm
from tests.test_gpu_block_norm import BF16, FP32, _check_forward, _check_gradients, _inputs

pytestmark = pytest.mark.gpu

KINDS = [dict(), dict(post=False), dict(y=False, post=False), dict(gate='channel'), dict(gate='token'), dict(gate='token', post=False), dict(gate='element')]
# one CTA a row, rows that are no whole groups of eight, two rows at a time, two CTAs a row
SHAPES = [(40, 512), (40, 250), (301, 2560), (5, 4104), (5, 5003)]


def _scaled(tokens, hidden, size, size_y, **kw):
    x, d_stream, d_normed = _inputs(tokens, hidden, **kw)
    x['residual'] = x['residual'] * size
    if x['y'] is not None:
        x['y'] = x['y'] * size_y
    return x, d_stream, d_normed


@pytest.mark.parametrize('tokens, hidden', SHAPES)
@pytest.mark.parametrize('types', [dict(dtype=FP32), dict(dtype=BF16), dict(dtype=BF16, stream=FP32)])
@pytest.mark.parametrize('size', [1e12, 1e14, 3e16])
def test_gradient_of_large_streams(tokens, hidden, types, size):
    """The part of the gradient that lies along the stream is as large as the rest of it, whatever the stream's size."""
    for i, kind in enumerate(KINDS):
        for size_y in (1.0, size):
            x, _, d_normed = _scaled(tokens, hidden, size, size_y, seed=i, **types, **kind)
            if x['y'] is None:
                d_normed = d_normed.to(x['residual'].dtype)
                x['pre_weight'] = x['pre_weight'].to(x['residual'].dtype)
            _check_gradients(x, None, d_normed, mm.block_norm_backward(None, d_normed, **x))


@pytest.mark.parametrize('tokens, hidden', SHAPES)
@pytest.mark.parametrize('types', [dict(dtype=FP32), dict(dtype=BF16)])
@pytest.mark.parametrize('size, eps', [(1e-10, 1e-28), (1e-15, 1e-30), (0.0, 1e-28), (0.0, 1e-34)])
def test_small_rows_and_small_eps(tokens, hidden, types, size, eps):
    """Rows whose mean square is far below 1, down to nothing but eps: the roots' powers leave the range of 32 bits, the gradients do not. A row of zeros beside ordinary rows
    does nothing to what is summed over the rows."""
    for i, kind in enumerate(KINDS):
        x, _, d_normed = _scaled(tokens, hidden, size, size, seed=i, **types, **kind)
        _check_forward(x, mm.block_norm(**x, eps=eps), eps=eps)
        _check_gradients(x, None, d_normed, mm.block_norm_backward(None, d_normed, **x, eps=eps), eps=eps)
        x, d_stream, d_normed = _inputs(tokens, hidden, seed=i, **types, **kind)
        for name in ('residual', 'y'):
            if x[name] is not None:
                x[name][tokens // 2:tokens // 2 + 2] = 0
        _check_gradients(x, d_stream, d_normed, mm.block_norm_backward(d_stream, d_normed, **x, eps=eps), eps=eps)


@pytest.mark.parametrize('size', [1.0, 1e-17, 1e-19, 1e-21, 0.0])
def test_smallest_eps(size):
    """Rows around the root of the smallest eps: squares below what 32 bits hold are nothing beside it."""
    for kind in (dict(), dict(gate='token')):
        x, _, _ = _scaled(20, 512, size, 1.0, dtype=FP32, **kind)
        x['post_weight'] = x['post_weight'] * size                         # the stream stays that small
        _check_forward(x, mm.block_norm(**x, eps=2.0 ** -126), eps=2.0 ** -126)
