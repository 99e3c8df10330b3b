"""The operators around the layer together, as a program uses them: a decode step, and a training step of a block."""
import pytest
import torch

import hopper_megamoe_basedondeepgemm_b200 as mm
from hopper_megamoe_basedondeepgemm_b200 import workload as W
from oracle import megamoe_oracle as O
from tests import util_block as B

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('tokens', [1, 24])
def test_block_around_the_layer(tokens):
    """Attention's output into the stream and normed in place, the layer from those hidden states, its output normed, gated and added: the same as the layer alone
    with plain norms around it."""
    experts, hidden, inter, fmt = 48, 1024, 512, 'mxfp4'
    g = torch.Generator(device='cuda').manual_seed(5)

    def randn(*shape):
        return torch.randn(shape, generator=g, device='cuda')
    stream, attn, gate = randn(tokens, hidden), randn(tokens, hidden).bfloat16(), torch.sigmoid(randn(tokens, 1)).bfloat16()
    w = [(1 + 0.1 * randn(hidden)).bfloat16() for _ in range(3)]
    router = (randn(experts, hidden) / hidden ** 0.5).bfloat16()
    l1, l2, _ = W.make_layer_weights(experts, hidden, inter, fmt, seed=3, std=0.05)
    buf = mm.get_symm_buffer_for_mega_moe(None, experts, 32, 8, hidden, inter, act_format=fmt)
    ws = torch.zeros(mm.fe_workspace_bytes(buf), dtype=torch.uint8, device='cuda')
    before, y = stream.clone(), torch.empty((tokens, hidden), dtype=torch.bfloat16, device='cuda')

    hid = torch.empty_like(attn)
    mm.block_norm(stream, attn, pre_weight=w[0], residual_out=stream, normed=hid)
    mm.mega_moe_from_hidden(y, hid, router, l1, l2, buf, ws, activation_clamp=10.0, timeout_ms=500.0)
    layer_out = y.clone()
    out, normed = mm.block_norm(stream, y, post_weight=w[1], pre_weight=w[2], gate=gate, residual_out=stream, normed=y)
    assert buf.device_status()[0] == 0 and out is stream and normed is y

    want, want_hid, size, size_hid = B.norm_reference(before, attn, w[0], None, None, 1.0, 1e-6, 0.0)
    B.assert_near(hid, want_hid, size_hid, 64, 'hidden states')
    first = before + attn.float()
    want, want_normed, size, size_normed = B.norm_reference(first, layer_out, w[2], w[1], gate, 1.0, 1e-6, 0.0)
    B.assert_near(stream, want, size, 64, 'stream')
    B.assert_near(normed, want_normed, size_normed, 64, 'normed')
    # and the layer from logits of the program's own (the frontend's: bf16, summed in its order), routed into the buffer's views
    logits = O.router_logits_device_order(hid.cpu(), router.cpu()).to(torch.bfloat16).cuda()
    idx, weights = buf.topk_idx[:tokens].clone(), buf.topk_weights[:tokens].clone()
    buf.topk_idx.zero_(), buf.topk_weights.zero_()
    mm.route_tokens(logits, 8, topk_idx=buf.topk_idx[:tokens], topk_weights=buf.topk_weights[:tokens])
    assert torch.equal(buf.topk_idx[:tokens], idx)
    assert torch.allclose(buf.topk_weights[:tokens], weights, rtol=2e-6, atol=1e-7)          # (the frontend's own tolerance)
    y2 = torch.empty_like(y)
    mm.fp4_fp4_mega_moe(y2, l1, l2, buf, activation_clamp=10.0, timeout_ms=500.0)
    assert buf.device_status()[0] == 0 and O.rel_rmse(y2.cpu(), layer_out.cpu()) <= 3e-3      # (the layer's parity bound)


@pytest.mark.parametrize('tokens', [1, 24])
def test_chain_without_a_pause(tokens):
    """Norm, layer, norm and routing of several blocks one behind the other, eager and as a graph: kernels that start before the ones ahead of them have ended find
    what those write. The same as with a wait after every call."""
    experts, hidden, inter, fmt, blocks = 48, 1024, 512, 'mxfp4', 4
    g = torch.Generator(device='cuda').manual_seed(8)

    def randn(*shape):
        return torch.randn(shape, generator=g, device='cuda')
    start, attn = randn(tokens, hidden), randn(tokens, hidden).bfloat16()
    w = (1 + 0.1 * randn(hidden)).bfloat16()
    router = (randn(experts, hidden) / hidden ** 0.5).bfloat16()
    l1, l2, _ = W.make_layer_weights(experts, hidden, inter, fmt, seed=3, std=0.05)
    buf = mm.get_symm_buffer_for_mega_moe(None, experts, 32, 8, hidden, inter, act_format=fmt)
    ws = torch.zeros(mm.fe_workspace_bytes(buf), dtype=torch.uint8, device='cuda')
    stream, hid, y, own = start.clone(), torch.empty_like(attn), torch.empty_like(attn), torch.empty((tokens, experts), device='cuda')

    def run(wait):
        seen = []
        stream.copy_(start)
        hid.copy_(attn)
        for _ in range(blocks):
            mm.block_norm(stream, hid, pre_weight=w, residual_out=stream, normed=hid)
            wait()
            mm.mega_moe_from_hidden(y, hid, router, l1, l2, buf, ws, activation_clamp=10.0, timeout_ms=500.0)
            wait()
            mm.block_norm(stream, y, post_weight=w, pre_weight=w, residual_out=stream, normed=hid)
            wait()
            torch.matmul(hid.float(), router.float().t(), out=own)
            wait()
            idx, weights = mm.route_tokens(own, 8, topk_idx=buf.topk_idx[:tokens], topk_weights=buf.topk_weights[:tokens])
            wait()
            b = mm.balance_loss(own, idx, z_coef=0.1)
            wait()
            d = mm.router_backward(own, idx, d_topk_weights=weights, balance=b)
            wait()
            mm.fp4_fp4_mega_moe(y, l1, l2, buf, activation_clamp=10.0, timeout_ms=500.0)
            wait()
            seen += [idx.clone(), b.counts, b.losses, d]
        return [stream.clone(), y.clone()] + seen
    want = run(torch.cuda.synchronize)
    for _ in range(3):
        got = run(lambda: None)
        torch.cuda.synchronize()
        assert buf.device_status()[0] == 0
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = run(lambda: None)
    for _ in range(3):
        for t in captured:
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert buf.device_status()[0] == 0
        assert all(torch.equal(a, b) for a, b in zip(captured, want))


class _Norm(torch.autograd.Function):
    """How a program hooks the pair into autograd."""

    @staticmethod
    def forward(ctx, residual, y, gate, pre, post):
        ctx.save_for_backward(residual, y, gate, pre, post)
        return mm.block_norm(residual, y, gate=gate, pre_weight=pre, post_weight=post)

    @staticmethod
    def backward(ctx, d_stream, d_normed):
        residual, y, gate, pre, post = ctx.saved_tensors
        g = mm.block_norm_backward(d_stream.contiguous(), d_normed.contiguous(), residual, y, gate=gate, pre_weight=pre, post_weight=post)
        return g.residual, g.y, g.gate, g.pre_weight, g.post_weight


class _Route(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, topk):
        idx, w = mm.route_tokens(logits, topk)
        b = mm.balance_loss(logits, idx, balance_coef=0.5, z_coef=0.1)
        ctx.save_for_backward(logits, idx)
        ctx.balance = b
        ctx.mark_non_differentiable(idx)
        return idx, w, b.loss

    @staticmethod
    def backward(ctx, _, d_w, d_loss):
        logits, idx = ctx.saved_tensors
        return mm.router_backward(logits, idx, d_topk_weights=d_w.contiguous(), balance=ctx.balance, d_loss=d_loss.contiguous()), None


def test_training_step_of_a_block():
    """Norm, router and balance loss of a block, hooked into autograd, against autograd through the plain forms in 64 bits. 32-bit tensors: what the
    chain adds up are roundings of 2^-24, a few hundred of them in a row of products and sums (the router's product has 256 terms)."""
    tokens, hidden, experts, topk = 60, 256, 48, 8
    g = torch.Generator(device='cuda').manual_seed(1)

    def randn(*shape):
        return torch.randn(shape, generator=g, device='cuda')
    leaves = [randn(tokens, hidden), randn(tokens, hidden), torch.sigmoid(randn(hidden)), 1 + 0.1 * randn(hidden), 1 + 0.1 * randn(hidden), randn(experts, hidden) / 16]
    d_stream, d_w = randn(tokens, hidden), randn(tokens, topk)
    a = [t.clone().requires_grad_(True) for t in leaves]
    stream, normed = _Norm.apply(*a[:5])
    idx, w, loss = _Route.apply(normed @ a[5].t(), topk)
    ((stream * d_stream).sum() + (w * d_w).sum() + loss).backward()

    b = [t.double().requires_grad_(True) for t in leaves]
    stream64, normed64, _, _ = B.norm_reference(b[0], b[1], b[3], b[4], b[2], 1.0, 1e-6, 0.0)
    logits64 = normed64 @ b[5].t()
    loss64 = B.balance_reference(logits64, idx, 0, None, 0.5, 0.1)[0][0]
    ((stream64 * d_stream.double()).sum() + (B.route_weights(logits64, idx, 0, 1.0) * d_w.double()).sum() + loss64).backward()
    loss, loss64 = loss.detach(), loss64.detach()
    assert abs(float(loss) - float(loss64)) <= 512 * B.U * float(loss64)
    for x, y in zip(a, b):
        assert float((x.grad.double() - y.grad).norm()) <= 512 * B.U * float(y.grad.norm())
