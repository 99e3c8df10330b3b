"""More of what the C ABI of the norms refuses: `mm_block_norm_backward` outputs that share memory with anything else of the call, weights' and gates' gradients and the workspace
among them, and an eps that 32 bits hold only in part."""
import ctypes

import pytest
import torch

from hopper_megamoe_basedondeepgemm_b200 import _lib
from tests.test_block_host import A, INVALID, _grads, _norm

W = 64 * 2                                    # bytes of a weight, and of a row, of 64 channels in bf16
NEED = 4 * 64 * 2 * 4                         # of the workspace: 4 CTAs, two sums of 64 channels in 32 bits
CHANNEL, TOKEN, ELEMENT = dict(gate=14 * A, gate_mode=1), dict(gate=14 * A, gate_mode=2, gate_stride=1), dict(gate=14 * A, gate_mode=3, gate_stride=64)


def _call(norm, grads):
    return _lib.load().mm_block_norm_backward(ctypes.byref(_norm(**norm)), ctypes.byref(_grads(**grads)), None)


@pytest.mark.parametrize('norm, grads', [
    ({}, dict(d_pre_weight=3 * A)), ({}, dict(d_post_weight=4 * A + W - 2)), ({}, dict(d_pre_weight=4 * A - W + 2)),                     # over weights
    ({}, dict(d_pre_weight=A)), ({}, dict(d_post_weight=2 * A + 3 * W)), ({}, dict(d_pre_weight=7 * A)), ({}, dict(d_post_weight=8 * A - 2)),   # over rows that are read
    ({}, dict(d_pre_weight=9 * A)), ({}, dict(d_post_weight=10 * A + 4 * W - 2)), ({}, dict(d_pre_weight=12 * A)), ({}, dict(d_post_weight=11 * A + 2)),      # over other outputs
    ({}, dict(workspace=A)), ({}, dict(workspace=3 * A)), ({}, dict(workspace=9 * A)), ({}, dict(workspace=11 * A)), ({}, dict(workspace=12 * A - NEED + 32)), ({}, dict(workspace=8 * A)),
    (CHANNEL, dict(d_gate=14 * A)), (CHANNEL, dict(d_gate=11 * A)), (CHANNEL, dict(d_gate=2 * A)), (CHANNEL, dict(d_gate=10 * A + 8)), (CHANNEL, dict(d_gate=13 * A + NEED - 2)),
    (CHANNEL, dict(d_gate=15 * A, workspace=14 * A)), (CHANNEL, dict(d_gate=15 * A, d_post_weight=14 * A + 2)),
    (TOKEN, dict(d_gate=12 * A, d_gate_stride=1)), (TOKEN, dict(d_gate=15 * A, d_gate_stride=1, workspace=15 * A - 32)), (ELEMENT, dict(d_gate=15 * A, d_pre_weight=15 * A + 3 * W)),
    (dict(tokens=0), dict(d_pre_weight=3 * A)), (dict(tokens=0), dict(d_pre_weight=12 * A)), (dict(tokens=0, **CHANNEL), dict(d_gate=4 * A)),
])
def test_overlaps_are_refused(norm, grads):
    assert _call(norm, grads) == INVALID


@pytest.mark.parametrize('norm, grads', [
    ({}, {}), ({}, dict(d_pre_weight=11 * A, d_post_weight=11 * A + W)), ({}, dict(workspace=12 * A + W)), (CHANNEL, dict(d_gate=14 * A + W)), (CHANNEL, dict(d_gate=13 * A + NEED)),
    (TOKEN, dict(d_gate=14 * A + 8, d_gate_stride=1)), (ELEMENT, dict(d_gate=14 * A + 4 * W)),
    (dict(pre_weight=3 * A, post_weight=3 * A), {}),                                                    # inputs may be one
    (dict(pre_weight=0, post_weight=0), dict(d_normed=0, d_pre_weight=0, d_post_weight=0, workspace=9 * A)),    # a workspace that is not needed is not looked at
])
def test_calls_that_pass_the_checks(norm, grads):
    """Without a GPU they get as far as asking for one."""
    if torch.cuda.is_available():
        pytest.skip('the addresses are not real')
    assert _call(norm, grads) == 3


@pytest.mark.parametrize('eps', [2.0 ** -127, 1e-40, 2.0 ** -149])
def test_subnormal_eps_is_refused(eps):
    """Beside such an eps the squares of small rows count, and 32 bits do not hold them."""
    assert _lib.load().mm_block_norm(ctypes.byref(_norm(eps=eps)), None) == INVALID
    assert _call(dict(eps=eps), {}) == INVALID


def test_smallest_eps():
    if torch.cuda.is_available():
        pytest.skip('the addresses are not real')
    assert _lib.load().mm_block_norm(ctypes.byref(_norm(eps=2.0 ** -126)), None) == 3 and _call(dict(eps=2.0 ** -126), {}) == 3
