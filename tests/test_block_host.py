"""Host side of the operators around the layer: what the C ABI and the Python functions refuse before anything is launched."""
import ctypes

import pytest
import torch

import hopper_megamoe_basedondeepgemm_b200 as mm
from hopper_megamoe_basedondeepgemm_b200 import _lib

INVALID, UNSUPPORTED = 1, 2
A = 1 << 20                                   # stand-in addresses, a MiB apart: nothing is read or written before the checks are through


def _norm(**kw):
    f = dict(residual=A, y=2 * A, gate=0, pre_weight=3 * A, post_weight=4 * A, residual_out=5 * A, normed=6 * A, tokens=4, residual_stride=64, y_stride=64,
             gate_stride=0, residual_out_stride=64, normed_stride=64, hidden=64, dtype=0, stream_dtype=0, weight_dtype=0, gate_dtype=0, gate_mode=0,
             scale=1.0, eps=1e-6, weight_offset=0.0)
    f.update(kw)
    a = _lib.MMBlockNormArgs()
    for k, v in f.items():
        setattr(a, k, v)
    return a


def _grads(**kw):
    f = dict(d_residual_out=7 * A, d_normed=8 * A, d_residual=9 * A, d_y=10 * A, d_gate=0, d_pre_weight=11 * A, d_post_weight=12 * A, d_residual_out_stride=64,
             d_normed_stride=64, d_residual_stride=64, d_y_stride=64, d_gate_stride=64, workspace=13 * A, workspace_bytes=1 << 20)
    f.update(kw)
    g = _lib.MMBlockNormGrads()
    for k, v in f.items():
        setattr(g, k, v)
    return g


def _router(**kw):
    f = dict(logits=A, topk_idx=2 * A, topk_weights=3 * A, logits_stride=48, tokens=4, num_experts=48, topk=8, dtype=2, score_mode=0, route_scale=1.0)
    f.update(kw)
    a = _lib.MMRouterArgs()
    for k, v in f.items():
        setattr(a, k, v)
    return a


def _balance(**kw):
    f = dict(cu_seqlens=4 * A, num_sequences=2, balance_coef=1.0, z_coef=0.1, counts=5 * A, seq_tokens=6 * A, mean_probs=7 * A, losses=8 * A)
    f.update(kw)
    b = _lib.MMBalanceArgs()
    for k, v in f.items():
        setattr(b, k, v)
    return b


def test_ctypes_mirror_matches_the_header():
    """Sizes and offsets of the structures in the ctypes mirror, as a C compiler sees them in the header."""
    import os
    import re
    import shutil
    import subprocess
    import tempfile
    if shutil.which('gcc') is None:
        pytest.skip('no C compiler')
    include = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), 'include')
    names = {'mm_block_norm_args_t': _lib.MMBlockNormArgs, 'mm_block_norm_grads_t': _lib.MMBlockNormGrads, 'mm_router_args_t': _lib.MMRouterArgs,
             'mm_balance_args_t': _lib.MMBalanceArgs}
    lines = [f'printf("%zu\\n", sizeof({c}));' + ''.join(f'printf("%zu\\n", offsetof({c}, {f[0]}));' for f in m._fields_) for c, m in names.items()]
    with tempfile.TemporaryDirectory() as d:
        with open(os.path.join(d, 'a.c'), 'w') as f:
            f.write('#include <stdio.h>\n#include <stddef.h>\n#include "megamoe_b200.h"\nint main(void) {' + '\n'.join(lines) + 'return 0; }')
        subprocess.run(['gcc', '-I', include, '-o', os.path.join(d, 'a'), os.path.join(d, 'a.c')], check=True)
        out = [int(v) for v in subprocess.run([os.path.join(d, 'a')], capture_output=True, text=True, check=True).stdout.split()]
    want = [v for m in names.values() for v in [ctypes.sizeof(m)] + [getattr(m, f[0]).offset for f in m._fields_]]
    assert out == want
    enums = re.findall(r'MM_(?:DTYPE|GATE)_\w+ = \d', open(os.path.join(include, 'megamoe_b200.h')).read())
    assert len(enums) == 7


@pytest.mark.parametrize('change, status', [
    (dict(tokens=-1), INVALID), (dict(tokens=(1 << 30) + 1), INVALID), (dict(hidden=0), INVALID), (dict(hidden=8193), UNSUPPORTED), (dict(dtype=3), INVALID), (dict(stream_dtype=-1), INVALID),
    (dict(stream_dtype=1), UNSUPPORTED), (dict(weight_dtype=1), UNSUPPORTED), (dict(gate_dtype=1), UNSUPPORTED), (dict(gate_mode=4), INVALID),
    (dict(gate_mode=1), INVALID), (dict(gate=14 * A), INVALID), (dict(y=0, residual_out=0), INVALID), (dict(y=0, residual_out=0, post_weight=0, pre_weight=0, normed=0), INVALID),
    (dict(eps=0.0), INVALID), (dict(eps=float('nan')), INVALID), (dict(scale=float('inf')), INVALID), (dict(weight_offset=float('nan')), INVALID),
    (dict(residual=0), INVALID), (dict(residual_out=0), INVALID), (dict(normed=0), INVALID), (dict(pre_weight=0), INVALID),
    (dict(residual_out_stride=63), INVALID), (dict(normed_stride=0), INVALID),
    (dict(residual_out=A + 2), INVALID), (dict(residual_out=A, residual_out_stride=65), INVALID), (dict(normed=5 * A), INVALID), (dict(normed=5 * A + 128), INVALID),
    (dict(normed=3 * A), INVALID), (dict(residual_out=4 * A - 64), INVALID),
    (dict(gate=14 * A, gate_mode=3, gate_stride=64, residual_out=14 * A), INVALID),
    (dict(residual_out=A, stream_dtype=2, residual=A + 128, residual_stride=64), INVALID),
])
def test_norm_refusals(change, status):
    assert _lib.load().mm_block_norm(ctypes.byref(_norm(**change)), None) == status


@pytest.mark.parametrize('change', [
    dict(), dict(tokens=1, residual_out_stride=0), dict(tokens=1, residual_out=A, residual_out_stride=7, normed=2 * A, normed_stride=1), dict(residual_out=A), dict(normed=2 * A), dict(normed=A), dict(residual_out=A, normed=2 * A),
    dict(residual=A, residual_out=A + 128, residual_stride=128, residual_out_stride=128),              # two halves of one buffer's rows
    dict(y=0, post_weight=0, residual_out=0), dict(pre_weight=0, normed=0),
])
def test_norm_calls_that_pass_the_checks(change):
    """Without a GPU they get as far as asking for one (with one they are not made here: the addresses are made up)."""
    if torch.cuda.is_available():
        pytest.skip('the addresses are not real')
    assert _lib.load().mm_block_norm(ctypes.byref(_norm(**change)), None) == 3


@pytest.mark.parametrize('norm, grads', [
    ({}, dict(d_normed=0)), ({}, dict(d_residual=0)), ({}, dict(d_y=0)), ({}, dict(d_pre_weight=0)), ({}, dict(d_post_weight=0)), ({}, dict(workspace=0)),
    ({}, dict(workspace_bytes=4 * 64 * 2 * 4 - 1)), ({}, dict(workspace=13 * A + 4)), ({}, dict(d_residual=7 * A)), ({}, dict(d_y=9 * A)), ({}, dict(d_y=A)),
    ({}, dict(d_residual=2 * A)), ({}, dict(d_y=3 * A)), ({}, dict(d_y_stride=63)), (dict(pre_weight=0), {}), (dict(y=0, post_weight=0), {}),
    (dict(gate=14 * A, gate_mode=1), {}), (dict(gate=14 * A, gate_mode=2, gate_stride=1), {}), (dict(gate=14 * A, gate_mode=3, gate_stride=64), dict(d_gate=14 * A)),
    (dict(gate=14 * A, gate_mode=3, gate_stride=64), dict(d_gate=9 * A)), (dict(eps=-1.0), {}), (dict(residual=0), {}),
])
def test_norm_gradient_refusals(norm, grads):
    assert _lib.load().mm_block_norm_backward(ctypes.byref(_norm(**norm)), ctypes.byref(_grads(**grads)), None) == INVALID
    assert _lib.load().mm_block_norm_backward(ctypes.byref(_norm()), None, None) == INVALID


def test_norm_workspace():
    lib = _lib.load()
    assert lib.mm_block_norm_workspace_bytes(-1, 64) == -1 and lib.mm_block_norm_workspace_bytes(4, 0) == -1 and lib.mm_block_norm_workspace_bytes(4, 8193) == -1
    assert lib.mm_block_norm_workspace_bytes(0, 64) == 0 and lib.mm_block_norm_workspace_bytes(1 << 40, 8192) < 1 << 26


@pytest.mark.parametrize('change, status', [
    (dict(tokens=-1), INVALID), (dict(num_experts=0), INVALID), (dict(num_experts=1025, logits_stride=1025), UNSUPPORTED), (dict(topk=0), INVALID), (dict(topk=33), UNSUPPORTED),
    (dict(num_experts=4), INVALID), (dict(dtype=5), INVALID), (dict(score_mode=2), INVALID), (dict(score_mode=-1), INVALID), (dict(logits=0), INVALID),
    (dict(topk_idx=0), INVALID), (dict(logits_stride=47), INVALID), (dict(tokens=(1 << 27) + 1), UNSUPPORTED),
])
def test_router_refusals(change, status):
    lib, a = _lib.load(), _router(**change)
    assert lib.mm_route_tokens(ctypes.byref(a), None, None, None) == status
    assert lib.mm_balance_loss(ctypes.byref(a), ctypes.byref(_balance()), 9 * A, 1 << 30, None) == status
    assert lib.mm_router_backward(ctypes.byref(a), None, ctypes.byref(_balance()), 1.0, None, 10 * A, 2048, None) == status


@pytest.mark.parametrize('change', [dict(num_sequences=0), dict(cu_seqlens=0), dict(counts=0), dict(seq_tokens=0), dict(balance_coef=float('nan')),
                                    dict(z_coef=float('inf')), dict(mean_probs=0), dict(losses=0)])
def test_balance_refusals(change):
    lib, a, b = _lib.load(), _router(), _balance(**change)
    assert lib.mm_balance_loss(ctypes.byref(a), ctypes.byref(b), 9 * A, 1 << 30, None) == INVALID
    if 'mean_probs' not in change and 'losses' not in change:
        assert lib.mm_router_backward(ctypes.byref(a), None, ctypes.byref(b), 1.0, None, 10 * A, 48, None) == INVALID


def test_router_refusals_of_its_other_arguments():
    lib, a, b = _lib.load(), _router(), _balance()
    assert lib.mm_route_tokens(ctypes.byref(a), 4 * A, None, None) == INVALID                          # a bias without sigmoid scores
    assert lib.mm_route_tokens(ctypes.byref(_router(topk_weights=0)), None, None, None) == INVALID
    assert lib.mm_route_tokens(ctypes.byref(_router(route_scale=float('nan'))), None, None, None) == INVALID
    need = lib.mm_balance_workspace_bytes(48, 2)
    assert lib.mm_balance_loss(ctypes.byref(a), ctypes.byref(b), 9 * A, need - 1, None) == INVALID
    assert lib.mm_balance_loss(ctypes.byref(a), ctypes.byref(b), 9 * A + 4, need, None) == INVALID
    assert lib.mm_balance_loss(ctypes.byref(a), ctypes.byref(b), None, need, None) == INVALID
    assert lib.mm_balance_workspace_bytes(48, (1 << 21) + 1) == -1 and lib.mm_balance_loss(ctypes.byref(a), ctypes.byref(_balance(num_sequences=(1 << 21) + 1)), 9 * A, 1 << 40, None) == UNSUPPORTED
    assert lib.mm_balance_workspace_bytes(0, 1) == -1 and lib.mm_balance_workspace_bytes(48, 0) == -1 and lib.mm_balance_workspace_bytes(1025, 1) == -1
    assert lib.mm_router_backward(ctypes.byref(a), None, None, 1.0, None, 10 * A, 48, None) == INVALID     # nothing to take the gradient of
    assert lib.mm_router_backward(ctypes.byref(a), 9 * A, None, 1.0, None, None, 48, None) == INVALID
    assert lib.mm_router_backward(ctypes.byref(a), 9 * A, None, 1.0, None, 10 * A, 47, None) == INVALID
    assert lib.mm_router_backward(ctypes.byref(a), 9 * A, None, 1.0, None, A + 64, 48, None) == INVALID    # over part of the logits


def test_router_outputs_lie_apart():
    """An output that shares memory with what the call reads, or with another output, is refused (first and last byte of 4 tokens of 48 experts, 8 routes)."""
    lib = _lib.load()
    logits, idx, weights = 4 * 48 * 4, 4 * 8 * 8, 4 * 8 * 4

    def route(bias=None, valid=None, **kw):
        return lib.mm_route_tokens(ctypes.byref(_router(score_mode=1, **kw)), bias, valid, None)
    for where in (A - 4, A, A + logits - 4, 2 * A - 4, 2 * A + idx - 4):
        assert route(topk_weights=where) == INVALID
    assert route(bias=2 * A + 8) == INVALID and route(bias=3 * A - 4) == INVALID and route(valid=3 * A + weights - 1) == INVALID and route(valid=2 * A - 3) == INVALID
    assert route(topk_idx=A + logits - 8) == INVALID

    need = lib.mm_balance_workspace_bytes(48, 2)

    def balance(workspace=9 * A, **kw):
        return lib.mm_balance_loss(ctypes.byref(_router()), ctypes.byref(_balance(**kw)), workspace, need, None)
    cells = 2 * 48 * 4
    for kw in (dict(counts=A), dict(mean_probs=2 * A + idx - 4), dict(seq_tokens=4 * A + 8), dict(losses=4 * A - 8), dict(counts=7 * A + cells - 4), dict(losses=6 * A + 4),
               dict(seq_tokens=5 * A - 4), dict(losses=9 * A + 8), dict(mean_probs=9 * A - 8), dict(workspace=2 * A), dict(workspace=8 * A + 8)):
        assert balance(**kw) == INVALID, kw

    def backward(d_logits, dw=9 * A, balance=True, d_loss=11 * A):
        return lib.mm_router_backward(ctypes.byref(_router()), dw, ctypes.byref(_balance()) if balance else None, 1.0, d_loss, d_logits, 48, None)
    for where in (2 * A, 2 * A + idx - 4, 9 * A, 9 * A + weights - 4, 4 * A + 8, 5 * A + cells - 4, 6 * A + 4, 11 * A - logits + 4, 11 * A):
        assert backward(where) == INVALID


def test_functions_take_gpu_tensors():
    x, w = torch.zeros(4, 64), torch.ones(64)
    with pytest.raises(RuntimeError):
        mm.block_norm(x, x, pre_weight=w)
    with pytest.raises(RuntimeError):
        mm.block_norm_backward(x, x, x, x, pre_weight=w)
    with pytest.raises(RuntimeError):
        mm.route_tokens(x, 8)
    with pytest.raises(RuntimeError):
        mm.balance_loss(x, torch.zeros(4, 8, dtype=torch.int64))
    with pytest.raises(RuntimeError):
        mm.router_backward(x, torch.zeros(4, 8, dtype=torch.int64), d_topk_weights=torch.zeros(4, 8))
