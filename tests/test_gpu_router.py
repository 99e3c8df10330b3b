"""`route_tokens`, `balance_loss` and `router_backward` on the GPU against plain forms in 64 bits (tolerances: util_block)."""
import pytest
import torch

import hopper_megamoe_basedondeepgemm_b200 as mm
from tests import util_block as B

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32
# A probability: an exponential (4 u) of a difference of logits (u of up to SPREAD of them), a sum of 32 in a lane and 5 steps over the warp, a
# reciprocal, a few products.
SPREAD = 40
CHAIN = SPREAD + 4 + 32 + 5 + 16
ROWS = 64                                      # probabilities that are added up in 32 bits


def _logits(tokens, experts, dtype=FP32, seed=0, width=1.5):
    g = torch.Generator(device='cuda').manual_seed(seed)
    return (torch.randn((tokens, experts), generator=g, device='cuda') * width).to(dtype)


def _bias(experts, seed=1):
    g = torch.Generator(device='cuda').manual_seed(seed)
    return torch.rand(experts, generator=g, device='cuda')


def _check_route(logits, topk, mode, bias, valid, scale, out):
    idx, w = B.route_reference(logits, topk, mode, bias, valid, scale)
    assert torch.equal(out[0], idx)
    B.assert_near(out[1], w, w.abs(), CHAIN, 'weights')


def _check_balance(logits, idx, mode, cu, a, z, b):
    l = logits.double()
    losses, counts, mean, tokens = B.balance_reference(l, idx, mode, cu, a, z)
    assert torch.equal(b.counts, counts) and torch.equal(b.tokens, tokens)
    # (a mean of n probabilities, each of which is kept to a multiple of 2^-36 after at most ROWS of them were added)
    B.assert_near(b.mean_probs, mean, mean + 2.0 ** -12, CHAIN + ROWS, 'mean_probs')
    lse = float(B.clean_logits(l)[B.clean_logits(l) > -float('inf')].abs().max()) if l.numel() else 0.0
    size = torch.stack([abs(a) * losses[1] + abs(z) * (losses[2] + lse), losses[1], losses[2] + lse])
    B.assert_near(b.losses, losses, size, 4 * (CHAIN + ROWS), 'losses')


def _check_gradient(logits, idx, mode, cu, a, z, scale, d_weights, d_loss, got):
    """The gradient by differentiation in 64 bits, and the magnitudes of the terms that make it up."""
    l = B.clean_logits(logits).requires_grad_(True)
    total = 0.0
    if a is not None:
        total = B.balance_reference(l, idx, mode, cu, a, z)[0][0] * d_loss
    if d_weights is not None:
        total = total + (B.route_weights(l, idx, mode, scale) * d_weights.double()).sum()
    total.backward()
    grad = l.grad if l.grad is not None else torch.zeros_like(l)
    t, e = logits.shape
    size = torch.zeros_like(grad)
    soft = torch.softmax(torch.where(torch.isnan(l.detach()), -float('inf'), l.detach()), dim=1).nan_to_num()
    p = soft
    if mode == 1:
        p = torch.where(l.detach() > -float('inf'), torch.sigmoid(l.detach()), 0.0)
        p = (p / p.sum(dim=1, keepdim=True)).nan_to_num()
    if a is not None:
        _, counts, _, n = B.balance_reference(l.detach(), idx, mode, cu, a, z)
        cuts = [0, t] if cu is None else cu.tolist()
        live, everyone = max(1, int((n > 0).sum())), max(1, int(n.sum()))
        top = l.detach().clamp(min=-1e30).amax(dim=1, keepdim=True)
        lse = top.abs() + 10.0
        for i, (lo, hi) in enumerate(zip(cuts[:-1], cuts[1:])):
            if hi <= lo:
                continue
            q = abs(a * d_loss) * counts[i].double() * e / (idx.shape[1] * max(1, int(n[i])) ** 2 * live)
            size[lo:hi] += p[lo:hi] * (q + (q * p[lo:hi]).sum(dim=1, keepdim=True)) + 2 * abs(z * d_loss) / everyone * lse[lo:hi] * soft[lo:hi]
    if d_weights is not None:
        w = B.route_weights(l.detach(), idx, mode, scale)
        dk = w * (d_weights.double().abs() + (w * d_weights.double().abs()).sum(dim=1, keepdim=True) / max(scale, 1e-30))
        size.scatter_add_(1, torch.where((idx >= 0) & (idx < e), idx, 0), dk)
    B.assert_near(got, grad, size, 4 * CHAIN, 'd_logits')


EXPERTS = [(1, 1), (7, 3), (32, 8), (33, 8), (48, 8), (64, 6), (100, 2), (128, 4), (250, 8), (256, 8), (384, 8), (511, 8), (512, 32), (640, 8), (1024, 8), (1023, 32)]


@pytest.mark.parametrize('experts, topk', EXPERTS)
@pytest.mark.parametrize('dtype', [FP32, BF16, FP16])
@pytest.mark.parametrize('mode', [0, 1])
def test_route(experts, topk, dtype, mode):
    for tokens, padded in ((1, False), (37, True), (600, False)):
        logits = _logits(tokens, experts, dtype, seed=tokens)
        bias = _bias(experts) if mode else None
        valid = (torch.arange(tokens, device='cuda') % 3 != 1) if padded else None
        out = mm.route_tokens(logits, topk, mode, bias, valid=valid, route_scale=2.5)
        _check_route(logits, topk, mode, bias, valid, 2.5, out)


@pytest.mark.parametrize('mode', [0, 1])
@pytest.mark.parametrize('experts', [40, 384, 1000])
def test_route_of_equal_keys(mode, experts):
    """Ties go to the lower expert: rows of one value, of two, sorted ones, and keys that differ by less than 32 bits tell."""
    logits = torch.zeros(9, experts, device='cuda')
    logits[1, ::2] = 1.0
    logits[2] = torch.arange(experts, device='cuda') // 7
    logits[3] = -(torch.arange(experts, device='cuda') // 7).float()
    logits[4] = 18.0 + torch.arange(experts, device='cuda') * 2.0 ** -16     # sigmoids that are all 1 in 32 bits, but not in 64
    logits[5] = torch.arange(experts, device='cuda') * 2.0 ** -30
    logits[6, -9:] = 3.0
    logits[7, 5:25] = torch.finfo(FP32).max
    logits[8] = torch.finfo(FP32).min
    _check_route(logits, 8, mode, None, None, 1.0, mm.route_tokens(logits, 8, mode))
    if mode:
        bias = torch.zeros(experts, device='cuda')
        bias[experts // 2:] = 2.0 ** -26
        _check_route(logits[:8], 8, mode, bias, None, 1.0, mm.route_tokens(logits[:8], 8, mode, bias))


def test_biases_of_any_size():
    """Biases that dwarf the scores (their keys' 32-bit errors are of another size than the border's), infinite ones, and -inf or NaN, which switch an expert off."""
    inf = float('inf')
    logits = _logits(300, 96)
    bias = _bias(96)
    for scale in (1e6, 1e30):
        big = bias.clone()
        big[::5] *= scale
        big[1::7] -= 3.0
        _check_route(logits, 8, 1, big, None, 1.0, mm.route_tokens(logits, 8, 1, big))
    bias[3:6] = inf
    _check_route(logits, 8, 1, bias, None, 1.0, mm.route_tokens(logits, 8, 1, bias))
    bias[10:90] = -inf
    bias[90:93] = float('nan')
    idx, w = mm.route_tokens(logits, 16, 1, bias)
    on = torch.cat([torch.arange(10), torch.arange(93, 96)]).cuda()
    want, _ = B.route_reference(logits[:, on].contiguous(), 13, 1, bias[on].contiguous(), None, 1.0)
    assert torch.equal(idx[:, :13], on[want]) and bool((idx[:, 13:] == -1).all()) and not w[:, 13:].any()


@pytest.mark.parametrize('mode', [0, 1])
def test_many_equal_keys(mode):
    """More candidates than a warp has lanes, and more routes than lanes with an expert on top."""
    logits = (_logits(64, 1024, seed=6) * 2).round()
    for topk in (1, 8, 32):
        _check_route(logits, topk, mode, None, None, 1.0, mm.route_tokens(logits, topk, mode))
    short = _logits(40, 40, seed=7)
    _check_route(short, 32, mode, None, None, 1.0, mm.route_tokens(short, 32, mode))


@pytest.mark.parametrize('mode', [0, 1])
def test_experts_that_are_off(mode):
    """-inf and NaN switch an expert off; rows with fewer experts left than routes, and with none; +inf; the type's lowest value is a value."""
    inf = float('inf')
    logits = _logits(8, 60)
    logits[0, 10:] = -inf
    logits[1, 3:] = float('nan')
    logits[2] = -inf
    logits[3, ::2] = float('nan')
    logits[4, 7] = inf
    logits[5, 5:] = torch.finfo(FP32).min
    logits[6, :59] = -inf
    out = mm.route_tokens(logits, 8, mode)
    _check_route(logits, 8, mode, None, None, 1.0, out)
    assert out[0][1].tolist()[3:] == [-1] * 5 and out[0][2].tolist() == [-1] * 8 and not out[1][2].any()
    finite = torch.tensor([0, 1, 2, 3, 6, 7], device='cuda')
    l, idx = logits[finite].contiguous(), out[0][finite].contiguous()
    b = mm.balance_loss(l, idx, mode, balance_coef=0.5, z_coef=0.1)
    _check_balance(l, idx, mode, None, 0.5, 0.1, b)
    dw = _logits(6, 8, seed=3)
    d = mm.router_backward(l, idx, mode, d_topk_weights=dw, balance=b, d_loss=2.0)
    _check_gradient(l, idx, mode, None, 0.5, 0.1, 1.0, dw, 2.0, d)
    assert not d[2].any() and not d[0, 10:].any()


@pytest.mark.parametrize('dtype', [FP32, BF16])
def test_large_logits(dtype):
    """Logits whose exponentials over- or underflow by themselves."""
    logits = torch.cat([_logits(20, 96, dtype, width=30.0), _logits(20, 96, dtype, seed=2) + 200.0, _logits(20, 96, dtype, seed=3) - 60.0]).contiguous()
    out = mm.route_tokens(logits, 8)
    idx, w = B.route_reference(logits, 8, 0, None, None, 1.0)
    assert torch.equal(out[0], idx)
    B.assert_near(out[1], w, w.abs(), CHAIN + 300, 'weights')
    out = mm.route_tokens(logits[20:].contiguous(), 8, 1)
    _check_route(logits[20:], 8, 1, None, None, 1.0, out)


def _sequences(tokens, n, seed=0):
    g = torch.Generator().manual_seed(seed)
    cuts = torch.sort(torch.randint(0, tokens + 1, (n + 1,), generator=g)).values
    cuts[0] = 0
    return cuts.int().cuda()


@pytest.mark.parametrize('experts, topk', EXPERTS)
@pytest.mark.parametrize('dtype', [FP32, BF16, FP16])
@pytest.mark.parametrize('mode', [0, 1])
def test_balance_and_gradient(experts, topk, dtype, mode):
    for tokens, sequences in ((1, 0), (3, 1), (150, 7), (700, 0)):
        logits = _logits(tokens, experts, dtype, seed=tokens)
        idx = mm.route_tokens(logits, topk, mode)[0]
        g = torch.Generator(device='cuda').manual_seed(tokens)
        idx[torch.rand(idx.shape, generator=g, device='cuda') < 0.1] = -1
        if tokens > 3:
            idx[5] = -1
            idx[6, 0] = experts                                   # outside of the experts: no route
            idx[7, -1] = idx[7, 0]                                # the same expert twice
        cu = _sequences(tokens, sequences) if sequences else None
        b = mm.balance_loss(logits, idx, mode, cu_seqlens=cu, balance_coef=0.3, z_coef=0.02)
        _check_balance(logits, idx, mode, cu, 0.3, 0.02, b)
        dw = _logits(tokens, topk, seed=4)
        d_loss = torch.full((), 1.7, device='cuda')
        d = mm.router_backward(logits, idx, mode, d_topk_weights=dw, route_scale=2.0, balance=b, d_loss=d_loss)
        _check_gradient(logits, idx, mode, cu, 0.3, 0.02, 2.0, dw, float(d_loss), d)
        _check_gradient(logits, idx, mode, cu, 0.3, 0.02, 1.0, None, 0.5, mm.router_backward(logits, idx, mode, balance=b, d_loss=0.5))
        _check_gradient(logits, idx, mode, None, None, None, 1.5, dw, None, mm.router_backward(logits, idx, mode, d_topk_weights=dw, route_scale=1.5))


@pytest.mark.parametrize('tokens, experts, sequences', [(20000, 48, 0), (383, 64, 32), (384, 64, 32), (385, 64, 32), (384, 64, 33), (384, 384, 5), (384, 385, 3), (384, 4, 511), (384, 4, 513), (9, 256, 8), (9000, 384, 3), (5000, 64, 600), (40, 16, 2000)])
@pytest.mark.parametrize('mode', [0, 1])
def test_many_tokens_and_sequences(tokens, experts, sequences, mode):
    logits = _logits(tokens, experts)
    idx = mm.route_tokens(logits, 4, mode)[0]
    cu = _sequences(tokens, sequences) if sequences else None
    b = mm.balance_loss(logits, idx, mode, cu_seqlens=cu, balance_coef=1.0, z_coef=0.01)
    _check_balance(logits, idx, mode, cu, 1.0, 0.01, b)
    d = mm.router_backward(logits, idx, mode, balance=b)
    _check_gradient(logits, idx, mode, cu, 1.0, 0.01, 1.0, None, 1.0, d)
    again = mm.balance_loss(logits, idx, mode, cu_seqlens=cu, balance_coef=1.0, z_coef=0.01)
    assert torch.equal(b.losses, again.losses) and torch.equal(b.mean_probs, again.mean_probs)      # whole-number sums
    assert torch.equal(d, mm.router_backward(logits, idx, mode, balance=again))


def test_tokens_behind_the_last_sequence():
    """They count nowhere and have no gradient of the loss; neither do sequences without routed tokens."""
    logits = _logits(50, 48)
    idx = mm.route_tokens(logits, 8)[0]
    idx[10:20] = -1
    cu = torch.tensor([0, 10, 20, 20, 33], dtype=torch.int32, device='cuda')
    b = mm.balance_loss(logits, idx, cu_seqlens=cu, z_coef=1.0)
    _check_balance(logits, idx, 0, cu, 1.0, 1.0, b)
    assert b.tokens.tolist() == [10, 0, 0, 13] and not b.counts[1:3].any() and not b.mean_probs[1:3].any()
    d = mm.router_backward(logits, idx, balance=b)
    assert not d[33:].any() and not d[10:20].any() and bool(d[:10].any())
    nothing = torch.full_like(idx, -1)
    b = mm.balance_loss(logits, nothing, cu_seqlens=cu, z_coef=1.0)
    assert not b.losses.any() and not b.counts.any() and not mm.router_backward(logits, nothing, balance=b).any()


def test_sequence_ends_of_any_content():
    """Ends that are not ascending, negative or beyond the tokens give some result, inside the tensors, and do no harm."""
    logits = _logits(64, 48)
    idx = mm.route_tokens(logits, 8)[0]
    for ends in ([0, 40, 20, 90, -7], [5, 5, 5], [-100, 2 ** 31 - 1], [70, 80], [2 ** 31 - 1, -2 ** 31]):
        cu = torch.tensor(ends, dtype=torch.int32, device='cuda')
        b = mm.balance_loss(logits, idx, cu_seqlens=cu)
        assert int(b.counts.sum()) == 8 * int(b.tokens.sum()) <= 64 * 8
        assert mm.router_backward(logits, idx, balance=b).isfinite().all()


@pytest.mark.parametrize('mode', [0, 1])
def test_no_tokens(mode):
    logits = torch.zeros(0, 48, device='cuda')
    idx, w = mm.route_tokens(logits, 8, mode)
    assert idx.shape == w.shape == (0, 8)
    b = mm.balance_loss(logits, idx, mode)
    assert not b.losses.any() and not b.counts.any() and not b.mean_probs.any() and b.tokens.tolist() == [0]
    assert mm.router_backward(logits, idx, mode, balance=b).shape == (0, 48)


@pytest.mark.parametrize('experts', [48, 50])
@pytest.mark.parametrize('dtype', [FP32, BF16])
def test_strided_logits(experts, dtype):
    """Logits and their gradient as columns of wider buffers, at aligned and odd places; in place."""
    for start, ld in ((0, 64), (3, 59), (8, 72)):
        buf = torch.full((100, ld), 9.0, dtype=dtype, device='cuda')
        logits = _logits(100, experts, dtype)
        buf[:, start:start + experts] = logits
        view = buf[:, start:start + experts]
        out = mm.route_tokens(view, 8)
        _check_route(logits, 8, 0, None, None, 1.0, out)
        b = mm.balance_loss(view, out[0])
        want = mm.router_backward(logits, out[0], balance=b)
        got = torch.full((100, ld), 5.0, dtype=dtype, device='cuda')
        d = mm.router_backward(view, out[0], balance=b, d_logits=got[:, start:start + experts])
        assert torch.equal(d, want) and bool((got[:, :start] == 5.0).all()) and bool((got[:, start + experts:] == 5.0).all())
        assert torch.equal(mm.router_backward(view, out[0], balance=b, d_logits=view), want) and torch.equal(view, want)


def test_logits_far_apart():
    """Element offsets beyond 32 bits."""
    ld = 2 ** 30 + 4
    buf = torch.empty(2 * ld + 48, dtype=FP32, device='cuda')
    far = torch.as_strided(buf, (3, 48), (ld, 1))
    logits = _logits(3, 48)
    far.copy_(logits)
    out = mm.route_tokens(far, 8)
    _check_route(logits, 8, 0, None, None, 1.0, out)
    b = mm.balance_loss(far, out[0])
    _check_balance(logits, out[0], 0, None, 1.0, 0.0, b)
    assert torch.equal(mm.router_backward(far, out[0], balance=b, d_logits=far), mm.router_backward(logits, out[0], balance=b))


def test_infinities_and_the_ends_of_the_range():
    """Rows with NaN, infinities and the largest numbers beside ordinary ones: losses and gradients of the ordinary rows are what they are without them."""
    inf, top = float('inf'), torch.finfo(FP32).max
    for mode in (0, 1):
        plain = _logits(12, 48)
        idx = mm.route_tokens(plain, 8, mode)[0]
        odd = plain.clone()
        odd[0, 3], odd[1, 4], odd[2, 5], odd[3], odd[4] = float('nan'), -inf, inf, top, -top
        odd[5] = -inf
        b = mm.balance_loss(odd, idx, mode)
        assert b.counts.sum() == 96 and b.losses[1].isfinite() and b.mean_probs.isfinite().all()
        p = torch.full((12, 48), 0.0, dtype=torch.float64, device='cuda')
        for r in range(12):
            l = B.clean_logits(odd[r:r + 1])[0]
            if bool((l > -inf).any()):
                s = torch.exp(l - l.max()) if mode == 0 else torch.where(l > -inf, torch.sigmoid(l), 0.0)
                p[r] = s / s.sum().clamp(min=1e-300)
        B.assert_near(b.mean_probs, p.mean(dim=0, keepdim=True), p.mean(dim=0, keepdim=True) + 2.0 ** -12, CHAIN + ROWS, 'mean_probs')
        whole = mm.balance_loss(plain, idx, mode)
        d, want = mm.router_backward(odd, idx, mode, balance=b), mm.router_backward(plain, idx, mode, balance=whole)
        assert torch.equal(d[6:], want[6:]) and not d[5].any()                # (the counts are the same)


def test_sums_over_ranks():
    """Counts and tokens of two halves of a batch, summed in between, give the gradient of the batch as a whole."""
    logits = _logits(90, 48)
    idx = mm.route_tokens(logits, 8)[0]
    whole = mm.balance_loss(logits, idx, balance_coef=0.5, z_coef=0.1)
    want = mm.router_backward(logits, idx, balance=whole)
    halves = [(logits[:40], idx[:40]), (logits[40:], idx[40:])]
    parts = [mm.balance_loss(l, i, balance_coef=0.5, z_coef=0.1) for l, i in halves]
    counts, tokens = parts[0].counts + parts[1].counts, parts[0].tokens + parts[1].tokens
    assert torch.equal(counts, whole.counts)
    for b in parts:
        b.counts.copy_(counts), b.tokens.copy_(tokens)
    assert torch.equal(torch.cat([mm.router_backward(l, i, balance=b) for (l, i), b in zip(halves, parts)]), want)


@pytest.mark.parametrize('tokens', [300, 2000])
def test_captured_and_replayed(tokens):
    """A training step's calls as a graph, replayed with new logits, two graphs at once."""
    logits, dw = _logits(tokens, 96), _logits(tokens, 8, seed=5)
    cu = _sequences(tokens, 6)

    def step(l):
        idx, w = mm.route_tokens(l, 8, 1, route_scale=2.0)
        b = mm.balance_loss(l, idx, 1, cu_seqlens=cu, balance_coef=0.1, z_coef=0.01)
        return idx, w, b.losses, b.counts, b.mean_probs, mm.router_backward(l, idx, 1, d_topk_weights=dw, route_scale=2.0, balance=b)
    step(logits)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step(logits)
        graphs.append((g, out))
    logits.copy_(_logits(tokens, 96, seed=8))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(3):
        for s, (g, _) in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    want = step(logits)
    for _, out in graphs:
        assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_two_streams_at_once():
    sets = [_logits(3000, 128, seed=s) for s in range(2)]
    idx = [mm.route_tokens(l, 8)[0] for l in sets]
    want = [mm.balance_loss(l, i, z_coef=0.1) for l, i in zip(sets, idx)]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(mm.balance_loss(sets[i], idx[i], z_coef=0.1))
    torch.cuda.synchronize()
    for i in range(2):
        for b in got[i]:
            assert torch.equal(b.losses, want[i].losses) and torch.equal(b.counts, want[i].counts) and torch.equal(b.mean_probs, want[i].mean_probs)


@pytest.mark.parametrize('mode', [0, 1])
def test_against_differences(mode):
    """The gradient against differences of the loss and of the weights along the gradient itself: a step of 2^-6 of a unit vector leaves under 2 %."""
    logits, dw = _logits(24, 48), _logits(24, 8, seed=5)
    idx = mm.route_tokens(logits, 8, mode)[0]

    def value(l):
        b = mm.balance_loss(l, idx, mode, balance_coef=3.0, z_coef=0.5)
        return float(b.losses[0].double()) + float((B.route_weights(l, idx, mode, 2.0) * dw.double()).sum())
    b = mm.balance_loss(logits, idx, mode, balance_coef=3.0, z_coef=0.5)
    d = mm.router_backward(logits, idx, mode, d_topk_weights=dw, route_scale=2.0, balance=b)
    way = d / d.norm()
    step = 2.0 ** -6
    slope = (value(logits + step * way) - value(logits - step * way)) / (2 * step)
    assert abs(slope - float(d.norm())) <= 0.02 * float(d.norm())


def test_refusals():
    l = _logits(8, 48)
    idx, _ = mm.route_tokens(l, 8)
    b = mm.balance_loss(l, idx)
    ones = torch.ones(48, device='cuda')
    bad = [
        lambda: mm.route_tokens(l[0], 8), lambda: mm.route_tokens(l.double(), 8), lambda: mm.route_tokens(l.cpu(), 8), lambda: mm.route_tokens(l.t(), 8),
        lambda: mm.route_tokens(l[:1].expand(8, 48), 8), lambda: mm.route_tokens(l, 0), lambda: mm.route_tokens(l, 33), lambda: mm.route_tokens(l[:, :4], 8),
        lambda: mm.route_tokens(torch.zeros(2, 1025, device='cuda'), 8), lambda: mm.route_tokens(l, 8, 2), lambda: mm.route_tokens(l, 8, 0, ones),
        lambda: mm.route_tokens(l, 8, 1, ones[:47]), lambda: mm.route_tokens(l, 8, 1, ones.half()), lambda: mm.route_tokens(l, 8, 1, ones.cpu()),
        lambda: mm.route_tokens(l, 8, valid=ones[:8]), lambda: mm.route_tokens(l, 8, valid=torch.ones(7, dtype=torch.bool, device='cuda')),
        lambda: mm.route_tokens(l, 8, route_scale=float('inf')), lambda: mm.route_tokens(l, 8, topk_idx=idx.int()), lambda: mm.route_tokens(l, 8, topk_idx=idx[:7]),
        lambda: mm.route_tokens(l, 8, topk_weights=torch.zeros(8, 16, device='cuda')[:, ::2]),
        lambda: mm.balance_loss(l, idx.int()), lambda: mm.balance_loss(l, idx[:7]), lambda: mm.balance_loss(l, idx.reshape(-1)), lambda: mm.balance_loss(l, idx.cpu()),
        lambda: mm.balance_loss(l, idx, cu_seqlens=torch.tensor([0, 8], device='cuda')), lambda: mm.balance_loss(l, idx, cu_seqlens=torch.tensor([0], dtype=torch.int32, device='cuda')),
        lambda: mm.balance_loss(l, idx, cu_seqlens=torch.tensor([0, 8], dtype=torch.int32)), lambda: mm.balance_loss(l, idx, z_coef=float('nan')),
        lambda: mm.router_backward(l, idx), lambda: mm.router_backward(l, idx, 1, balance=b), lambda: mm.router_backward(l[:, :40], idx, balance=b),
        lambda: mm.router_backward(l, idx, d_topk_weights=l), lambda: mm.router_backward(l, idx, balance=b, d_loss=ones), lambda: mm.router_backward(l, idx, balance=b, d_loss=torch.ones(())),
        lambda: mm.router_backward(l, idx, balance=b, d_logits=l.half()), lambda: mm.router_backward(l[:4], idx[:4], balance=b, d_logits=l[1:5]),
        lambda: mm.router_backward(l, idx.reshape(-1), balance=b), lambda: mm.router_backward(l, idx, balance=b, d_logits=torch.zeros(48, 8, device='cuda').t()),
    ]
    for i, f in enumerate(bad):
        with pytest.raises(RuntimeError):
            f()
            print('not refused:', i)


@pytest.mark.parametrize('mode', [0, 1])
def test_same_routes_as_the_frontend(mode):
    """`fe_forward_into_buffer` routes from hidden states; from its logits `route_tokens` gives the same experts and weights. (Hidden states and router
    weights of few bits: the sums are exact in 32 bits whatever their order, and the frontend rounds them once, to bf16.)"""
    tokens, experts, hidden = 40, 48, 512
    g = torch.Generator(device='cuda').manual_seed(0)
    x = torch.randint(-4, 5, (tokens, hidden), generator=g, device='cuda').to(BF16)
    wr = (torch.randint(-4, 5, (experts, hidden), generator=g, device='cuda').float() / 64).to(BF16)
    buf = mm.get_symm_buffer_for_mega_moe(None, experts, 64, 8, hidden, 256, act_format='mxfp4')
    ws = torch.zeros(mm.fe_workspace_bytes(buf), dtype=torch.uint8, device='cuda')
    bias = _bias(experts) if mode else None
    mm.fe_forward_into_buffer(x, wr, buf, ws, score_mode=mode, expert_bias=bias)
    logits = (x.double() @ wr.double().t()).to(BF16)
    idx, w = mm.route_tokens(logits, 8, mode, bias)
    apart = torch.ones(tokens, dtype=torch.bool, device='cuda')
    if mode:                                                               # (the frontend compares its keys in 32 bits)
        key = torch.sort(torch.sigmoid(logits.double()) + bias.double(), dim=1, descending=True).values
        apart = (key[:, :8] - key[:, 1:9]).amin(dim=1) > 2.0 ** -20
    assert int(apart.sum()) > tokens // 2
    assert torch.equal(idx[apart], buf.topk_idx[:tokens][apart])
    B.assert_near(buf.topk_weights[:tokens][apart], w[apart].double(), w[apart].double(), 2 * CHAIN, 'weights')
