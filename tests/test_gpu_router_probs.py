"""Mean probabilities of experts that a router hardly ever looks at (plain forms and tolerances: test_gpu_router, util_block)."""
import pytest
import torch

import hopper_megamoe_basedondeepgemm_b200 as mm
from tests import util_block as B
from tests.test_gpu_router import CHAIN, ROWS, _logits, _sequences

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('tokens, experts, sequences', [(1, 600, 0), (300, 48, 3), (700, 48, 0), (700, 48, 9), (900, 640, 4), (20000, 64, 0), (6000, 300, 40)])
@pytest.mark.parametrize('mode', [0, 1])
def test_small_probabilities(tokens, experts, sequences, mode):
    """Each to 32 bits of its own, or to the step of the sums: experts whose logits lie 8 to 32 below the others'. Sums are kept to multiples of 2^-63 of the tokens' next power
    of two, half of which every warp's part may be off by; a part has a token at least, so that much a mean. (A part of less than half a step is 0, so a mean can be; where the
    mean is a step, some part is one.)"""
    logits = _logits(tokens, experts, seed=tokens)
    logits[:, ::3] -= torch.linspace(8, 32, (experts + 2) // 3, device='cuda')
    idx = mm.route_tokens(logits, 4, mode)[0]
    cu = _sequences(tokens, sequences) if sequences else None
    b = mm.balance_loss(logits, idx, mode, cu_seqlens=cu)
    mean = B.balance_reference(logits.double(), idx, mode, cu, 1.0, 0.0)[2]
    step = 2.0 ** ((tokens - 1).bit_length() - 63)
    B.assert_near(b.mean_probs, mean, mean + step / 2 / (B.U * (CHAIN + ROWS)), CHAIN + ROWS, 'mean_probs')
    assert bool((b.mean_probs[mean >= step] > 0).all()) and not b.mean_probs[b.tokens == 0].any()
