"""The router's calls one behind the other over the same buffers, whose contents change from turn to turn, without a wait in between."""
import pytest
import torch

import hopper_megamoe_basedondeepgemm_b200 as mm

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('tokens, experts, sequences', [(6000, 96, 0), (6000, 96, 20), (3000, 256, 40), (500, 640, 3), (300, 48, 5)])
@pytest.mark.parametrize('mode', [0, 1])
def test_buffers_that_change_from_turn_to_turn(tokens, experts, sequences, mode):
    """Logits by torch's kernels or in the gradient's place, routes into one buffer: the same as with a wait after every call."""
    turns = 6
    g = torch.Generator(device='cuda').manual_seed(3)
    given = [torch.randn((tokens, experts), generator=g, device='cuda') * 2 for _ in range(turns)]
    cu = torch.sort(torch.randint(0, tokens + 1, (sequences + 1,), generator=g, device='cuda')).values.int() if sequences else None
    logits, idx, weights = torch.empty_like(given[0]), torch.zeros((tokens, 8), dtype=torch.int64, device='cuda'), torch.zeros((tokens, 8), device='cuda')

    def run(wait):
        seen = []
        for i in range(turns):
            logits.copy_(given[i])
            for _ in range(2):
                mm.route_tokens(logits, 8, mode, topk_idx=idx, topk_weights=weights)
                wait()
                b = mm.balance_loss(logits, idx, mode, cu_seqlens=cu, z_coef=0.1)
                wait()
                seen += [b.losses, b.counts, b.mean_probs, b.tokens, idx.clone()]
                wait()
                # the gradient over the logits, which are the next calls' logits
                mm.router_backward(logits, idx, mode, d_topk_weights=weights, balance=b, d_loss=1e4, d_logits=logits)
                wait()
        return seen + [logits.clone()]
    want = run(torch.cuda.synchronize)
    for _ in range(3):
        got = run(lambda: None)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = run(lambda: None)
    for _ in range(2):
        for t in captured:
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(captured, want))
