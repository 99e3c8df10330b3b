"""The operators around the expert-parallel layer, as cases that can be timed and compared with their plain forms.

Two families, each through the package's public functions:

  the norms of a transformer block, fused with its gate and the residual stream   `block_norm`, `block_norm_backward`
  routing from logits, the balance loss and the gradient of both                   `route_tokens`, `balance_loss`, `router_backward`

`listed()` are the standing cases, `draw(rng)` gives more of the same ranges. With `own` false `run` computes the plain form with
elementary torch operations in 32 bits (64 where keys lie next to a border, or sums are long), with `own` true it calls the package.

A case is a dict of plain values:

  path      'norm'         residual stream and a block's output -> new stream and the next block's input
            'norm grad'    gradients of those two -> gradients of stream, output, gate and weights
            'route'        logits -> expert ids and weights
            'balance'      logits and expert ids -> balance loss, z loss, counts, mean probabilities, and the logits' gradient
            'router step'  'route' and 'balance' of a training step together, with the gradient through the routing weights
  dtype     of the block's output, the normed rows and the gate; for the router of the logits
  stream    dtype of the residual stream
  tokens, hidden           rows and channels
  post, pre                norm of the block's output, norm of the new stream
  gate      'none', 'channel' [H], 'token' [T, 1] or 'element' [T, H]
  scale, offset            residual scale; weights count as offset + w
  experts, topk            of the router
  scores    'softmax', or 'sigmoid' with a Zipf(1.2) expert bias
  padded    share of the tokens that are padding;  dropped: share of routing slots that are switched off
  sequences 0: the batch as a whole, else ragged sequences, with some tokens behind the last one
"""
import math

import numpy as np
import torch

own = False

DTYPES = {'bf16': torch.bfloat16, 'fp16': torch.float16, 'fp32': torch.float32}
EPS = 1e-6
BALANCE, Z = 1e-2, 1e-3                      # coefficients of the two losses
ROUTE_SCALE = 2.5                            # of the routing weights, sigmoid scores
LARGEST_BYTES = 16384 * 4096 * 12            # of the largest listed case


def _norm(name, path, tokens, hidden, dtype, stream, post, pre, gate, scale=1.0, offset=0.0):
    c = dict(path=path, tokens=tokens, hidden=hidden, dtype=dtype, stream=stream, post=post, pre=pre, gate=gate, scale=scale, offset=offset)
    return dict(name=name, **c) if name else c


def _router(name, path, tokens, experts, topk, dtype, scores, padded=0.0, dropped=0.0, sequences=0):
    c = dict(path=path, tokens=tokens, experts=experts, topk=topk, dtype=dtype, scores=scores, padded=padded, dropped=dropped, sequences=sequences)
    return dict(name=name, **c) if name else c


def listed():
    return [
        # decode of one request: both norms of a block between attention and the layer
        _norm('norm, 1 token', 'norm', 1, 3072, 'bf16', 'bf16', True, True, 'none'),
        # a ragged batch of an odd width, each token's output gated by a scalar (a shared expert's gate)
        _norm('norm, 333 of 1001, fp16', 'norm', 333, 1001, 'fp16', 'fp16', False, True, 'token', scale=0.5),
        # the largest prefill: stream kept in 32 bits, a learned gate per channel
        _norm('norm, 16384 of 4096', 'norm', 16384, 4096, 'bf16', 'fp32', True, True, 'channel', offset=1.0),
        # a small training batch in 32 bits, gate per element
        _norm('norm grad, 100 of 1024, fp32', 'norm grad', 100, 1024, 'fp32', 'fp32', True, True, 'element', scale=0.7),
        # an ordinary micro-batch, plain pre-norm block
        _norm('norm grad, 2500 of 2048', 'norm grad', 2500, 2048, 'bf16', 'fp32', False, True, 'channel'),
        # a large one, norms on both sides
        _norm('norm grad, 8192 of 3072', 'norm grad', 8192, 3072, 'bf16', 'bf16', True, True, 'token'),
        # decode of one request over the experts of one rank
        _router('route, 1 of 48', 'route', 1, 48, 8, 'fp32', 'softmax'),
        # a prefill chunk over eight ranks' experts, biased sigmoid scores, some padding
        _router('route, 8192 of 384', 'route', 8192, 384, 8, 'fp32', 'sigmoid', padded=0.05),
        # a few short sequences over the experts of one rank, 16-bit logits
        _router('balance, 300 of 48, bf16', 'balance', 300, 48, 8, 'bf16', 'softmax', dropped=0.05, sequences=5),
        # one large micro-batch balanced as a whole
        _router('balance, 16384 of 384', 'balance', 16384, 384, 8, 'fp32', 'softmax'),
        # many ragged sequences, each balanced by itself
        _router('balance, 12000 of 128', 'balance', 12000, 128, 4, 'fp32', 'sigmoid', padded=0.1, sequences=37),
        # all that a training step asks of the router
        _router('router step, 4096 of 256', 'router step', 4096, 256, 8, 'fp32', 'sigmoid', padded=0.02, sequences=9),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    path = rng.choice(['norm', 'norm', 'norm grad', 'norm grad', 'route', 'balance', 'balance', 'router step'])
    tokens = _log_int(rng, 1, 16384)
    if path in ('norm', 'norm grad'):
        hidden = rng.choice([512 * rng.randint(1, 8), 8 * _log_int(rng, 8, 512), _log_int(rng, 64, 4096)])
        dtype = rng.choice(['bf16', 'bf16', 'fp16', 'fp32'])
        stream = rng.choice([dtype, 'fp32'])
        post, pre = rng.choice([(True, True), (True, True), (False, True), (True, False), (False, False)])
        gate = rng.choice(['none', 'channel', 'token', 'element'])
        c = _norm(None, path, tokens, hidden, dtype, stream, post, pre, gate, scale=rng.choice([1.0, round(rng.uniform(0.1, 2.0), 3)]), offset=rng.choice([0.0, 1.0]))
        while work(c)['bytes'] > LARGEST_BYTES:
            c['tokens'] = c['tokens'] // 2
        return c
    experts = _log_int(rng, 8, 512)
    return _router(None, path, tokens, experts, rng.choice([k for k in (1, 2, 4, 6, 8) if k <= experts]), rng.choice(['fp32', 'fp32', 'bf16', 'fp16']),
                   rng.choice(['softmax', 'sigmoid']), padded=rng.choice([0.0, 0.1]), dropped=rng.choice([0.0, 0.05]) if path == 'balance' else 0.0,
                   sequences=0 if path == 'route' else rng.choice([0, 0, min(tokens, _log_int(rng, 1, 64))]))


def _gate_shape(c):
    t, h = c['tokens'], c['hidden']
    return {'channel': (h,), 'token': (t, 1), 'element': (t, h)}[c['gate']]


def _prepare_norm(c, g):
    t, h, dtype = c['tokens'], c['hidden'], DTYPES[c['dtype']]

    def randn(*shape):
        return torch.randn(shape, generator=g, device='cuda')
    # a residual stream has a few channels that are far larger than the others
    channels = torch.exp(0.5 * randn(h)) * torch.where(torch.rand(h, generator=g, device='cuda') < 0.01, 8.0, 1.0)
    s = dict(case=c, residual=(randn(t, h) * channels).to(DTYPES[c['stream']]), y=randn(t, h).to(dtype), gate=None, post=None, pre=None)
    if c['gate'] != 'none':
        s['gate'] = torch.sigmoid(randn(*_gate_shape(c))).to(dtype)
    for name in ('post', 'pre'):
        if c[name]:
            s[name] = (1.0 - c['offset'] + 0.2 * randn(h)).to(dtype)
    if c['path'] == 'norm grad':
        s['d_stream'] = randn(t, h).to(DTYPES[c['stream']])
        s['d_normed'] = randn(t, h).to(dtype) if c['pre'] else None
    return s


def _prepare_router(c, g):
    t, e = c['tokens'], c['experts']

    def rand(*shape):
        return torch.rand(shape, generator=g, device='cuda')
    # logits of a router that has learned something: a common offset per expert and a spread per token
    logits = (torch.randn((t, e), generator=g, device='cuda') * 1.5 + torch.randn((1, e), generator=g, device='cuda') * 0.5).to(DTYPES[c['dtype']])
    s = dict(case=c, logits=logits, bias=None, valid=None, cu_seqlens=None, d_loss=1.0 / 3.0)
    if c['scores'] == 'sigmoid':
        s['bias'] = (1.0 / torch.arange(1, e + 1, dtype=torch.float32, device='cuda') ** 1.2)[torch.randperm(e, generator=g, device='cuda')].contiguous()
    if c['padded'] > 0:
        s['valid'] = rand(t) >= c['padded']
    if c['sequences']:
        # ragged sequences; what lies behind the last one is not part of the batch
        cuts = (rand(c['sequences'] + 1) * (t + 1)).floor().clamp(max=t).int().sort().values
        cuts[0] = 0
        s['cu_seqlens'] = cuts.contiguous()
    if c['path'] == 'balance':
        idx, _ = _plain_route(s)
        s['topk_idx'] = idx.masked_fill(rand(t, c['topk']) < c['dropped'], -1).contiguous()
    if c['path'] == 'router step':
        s['d_weights'] = torch.randn((t, c['topk']), generator=g, device='cuda') * 1e-3
    return s


def prepare(case, seed):
    g = torch.Generator(device='cuda').manual_seed(seed)
    return _prepare_norm(case, g) if case['path'] in ('norm', 'norm grad') else _prepare_router(case, g)


# ---------------------------------------------------------------- plain forms

def _rms(x):
    return torch.rsqrt((x * x).mean(dim=-1, keepdim=True) + EPS)


def _plain_norm(s):
    c = s['case']
    u = s['y'].float()
    if s['post'] is not None:
        u = u * _rms(u) * (s['post'].float() + c['offset'])
    if s['gate'] is not None:
        u = u * s['gate'].float()
    stream = s['residual'].float() + c['scale'] * u
    normed = None
    if s['pre'] is not None:
        normed = (stream * _rms(stream) * (s['pre'].float() + c['offset'])).to(s['y'].dtype)
    return {'stream': stream.to(s['residual'].dtype), 'normed': normed}


def _plain_norm_grad(s):
    c, dtype = s['case'], s['y'].dtype
    y = s['y'].float()
    gate = s['gate'].float() if s['gate'] is not None else None
    n1 = y
    if s['post'] is not None:
        i1, w1 = _rms(y), s['post'].float() + c['offset']
        n1 = y * i1
        u = n1 * w1
    else:
        u = y
    d_stream = s['d_stream'].float()
    out = {'gate': None, 'post': None, 'pre': None}
    if s['pre'] is not None:
        stream = s['residual'].float() + c['scale'] * (u if gate is None else u * gate)
        i2, w2, d_normed = _rms(stream), s['pre'].float() + c['offset'], s['d_normed'].float()
        n2, d_n2 = stream * i2, d_normed * w2
        d_stream = d_stream + i2 * (d_n2 - n2 * (d_n2 * n2).mean(dim=-1, keepdim=True))
        out['pre'] = (d_normed * n2).sum(dim=0).to(dtype)
    d_v = c['scale'] * d_stream
    d_u = d_v
    if gate is not None:
        d_gate = d_v * u
        if c['gate'] == 'channel':
            d_gate = d_gate.sum(dim=0)
        elif c['gate'] == 'token':
            d_gate = d_gate.sum(dim=1, keepdim=True)
        out['gate'] = d_gate.to(dtype)
        d_u = d_v * gate
    d_y = d_u
    if s['post'] is not None:
        d_n1 = d_u * w1
        d_y = i1 * (d_n1 - n1 * (d_n1 * n1).mean(dim=-1, keepdim=True))
        out['post'] = (d_u * n1).sum(dim=0).to(dtype)
    out['residual'], out['y'] = d_stream.to(s['residual'].dtype), d_y.to(dtype)
    return out


def _plain_weights(s, l, idx):
    """Routing weights over a row's routed slots, without their scale, and what is needed of the scores for the gradient."""
    live = idx >= 0
    chosen = l.gather(1, idx.clamp(min=0))
    if s['bias'] is None:
        chosen = chosen.masked_fill(~live, -math.inf)
        top = chosen.amax(dim=1, keepdim=True)
        scores = torch.exp(chosen - torch.where(top > -math.inf, top, 0.0))
    else:
        scores = (1.0 / (1.0 + torch.exp(-chosen))).masked_fill(~live, 0.0)
    total = scores.sum(dim=1, keepdim=True)
    return scores / torch.where(total > 0, total, 1.0), scores, torch.where(total > 0, total, 1.0)


def _route_scale(s):
    return 1.0 if s['bias'] is None else ROUTE_SCALE


def _plain_route(s):
    l = s['logits'].float()
    # the keys of two experts can lie closer than 32 bits tell: they are compared in 64
    keys = l.double()
    if s['bias'] is not None:
        keys = 1.0 / (1.0 + torch.exp(-keys)) + s['bias'].double()
    keys = torch.where(l > -math.inf, keys, -math.inf)               # (NaN and -inf: an expert that is switched off)
    keys, idx = torch.sort(keys, dim=1, descending=True, stable=True)
    k = s['case']['topk']
    idx = torch.where(keys[:, :k] > -math.inf, idx[:, :k], -1)
    if s['valid'] is not None:
        idx = torch.where(s['valid'][:, None], idx, -1)
    return idx, _plain_weights(s, l, idx)[0] * _route_scale(s)


def _segments(s):
    """Each token's sequence (the number of sequences: in none), and how many there are."""
    t = s['case']['tokens']
    if s['cu_seqlens'] is None:
        return torch.zeros(t, dtype=torch.int64, device='cuda'), 1
    n = s['cu_seqlens'].numel() - 1
    return torch.bucketize(torch.arange(t, device='cuda'), s['cu_seqlens'][1:].long(), right=True), n


def _plain_balance(s, idx, d_weights=None):
    c = s['case']
    t, e, k = c['tokens'], c['experts'], c['topk']
    l = s['logits'].float()
    segment, n = _segments(s)
    routed = (idx >= 0).any(dim=1) & (segment < n)
    member = ((segment[None, :] == torch.arange(n, device='cuda')[:, None]) & routed[None, :]).double()
    top = l.amax(dim=1, keepdim=True)
    ex = torch.exp(l - top)
    total = ex.sum(dim=1, keepdim=True)
    softmax, lse = ex / total, (top + torch.log(total))
    if s['bias'] is None:
        p = softmax
    else:
        scores = 1.0 / (1.0 + torch.exp(-l))
        p = scores / scores.sum(dim=1, keepdim=True)
    slots = torch.zeros((t, e + 1), dtype=torch.float64, device='cuda')
    slots.scatter_add_(1, torch.where(idx >= 0, idx, e), torch.ones_like(idx, dtype=torch.float64))
    tokens = member.sum(dim=1)
    counts = member @ slots[:, :e]
    mean = (member @ p.double()) / tokens.clamp(min=1.0)[:, None]
    load = counts * e / (k * tokens.clamp(min=1.0))[:, None]
    live, everyone = (tokens > 0).sum().clamp(min=1).double(), tokens.sum().clamp(min=1.0)
    balance = (load * mean).sum() / live
    z = torch.where(routed, lse[:, 0].double() ** 2, 0.0).sum() / everyone
    losses = torch.stack([BALANCE * balance + Z * z, balance, z]).float()
    # gradient: through p for the balance, through the logarithm of the sum for z
    q = (BALANCE * s['d_loss'] * load / (tokens.clamp(min=1.0) * live)[:, None]).float()[segment.clamp(max=n - 1)]
    inner = (q * p).sum(dim=1, keepdim=True)
    d = p * (q - inner)
    if s['bias'] is not None:
        d = d * (1.0 - scores)
    d = d + (2.0 * Z * s['d_loss'] / everyone).float() * lse * softmax
    d = torch.where(routed[:, None], d, 0.0)
    if d_weights is not None:
        w, chosen, of = _plain_weights(s, l, idx)
        dw = d_weights * _route_scale(s)
        dk = w * (dw - (w * dw).sum(dim=1, keepdim=True))
        if s['bias'] is not None:
            dk = dk * (1.0 - chosen)
        wide = torch.zeros((t, e + 1), dtype=torch.float32, device='cuda')
        d = d + wide.scatter_add_(1, torch.where(idx >= 0, idx, e), dk)[:, :e]
    return {'losses': losses, 'counts': counts.int(), 'mean_probs': mean.float(), 'tokens': tokens.int(), 'd_logits': d.to(s['logits'].dtype)}


# ---------------------------------------------------------------- one pass

def _own(s):
    import hopper_megamoe_basedondeepgemm_b200 as mm
    c = s['case']
    if c['path'] == 'norm':
        stream, normed = mm.block_norm(s['residual'], s['y'], pre_weight=s['pre'], post_weight=s['post'], gate=s['gate'], scale=c['scale'],
                                       eps=EPS, weight_offset=c['offset'])
        return {'stream': stream, 'normed': normed}
    if c['path'] == 'norm grad':
        g = mm.block_norm_backward(s['d_stream'], s['d_normed'], s['residual'], s['y'], pre_weight=s['pre'], post_weight=s['post'], gate=s['gate'],
                                   scale=c['scale'], eps=EPS, weight_offset=c['offset'])
        return {'residual': g.residual, 'y': g.y, 'gate': g.gate, 'post': g.post_weight, 'pre': g.pre_weight}
    mode = 0 if s['bias'] is None else 1
    if c['path'] == 'balance':
        b = mm.balance_loss(s['logits'], s['topk_idx'], score_mode=mode, cu_seqlens=s['cu_seqlens'], balance_coef=BALANCE, z_coef=Z)
        d = mm.router_backward(s['logits'], s['topk_idx'], score_mode=mode, balance=b, d_loss=s['d_loss'])
        return {'losses': b.losses, 'counts': b.counts, 'mean_probs': b.mean_probs, 'tokens': b.tokens, 'd_logits': d}
    idx, w = mm.route_tokens(s['logits'], c['topk'], score_mode=mode, expert_bias=s['bias'], valid=s['valid'], route_scale=_route_scale(s))
    if c['path'] == 'route':
        return {'idx': idx, 'weights': w}
    b = mm.balance_loss(s['logits'], idx, score_mode=mode, cu_seqlens=s['cu_seqlens'], balance_coef=BALANCE, z_coef=Z)
    d = mm.router_backward(s['logits'], idx, score_mode=mode, d_topk_weights=s['d_weights'], route_scale=_route_scale(s), balance=b, d_loss=s['d_loss'])
    return {'idx': idx, 'weights': w, 'losses': b.losses, 'counts': b.counts, 'mean_probs': b.mean_probs, 'tokens': b.tokens, 'd_logits': d}


def _given(d):
    return {k: v for k, v in d.items() if v is not None}


def run(s):
    if own:
        return _given(_own(s))
    path = s['case']['path']
    if path == 'norm':
        return _given(_plain_norm(s))
    if path == 'norm grad':
        return _given(_plain_norm_grad(s))
    if path == 'balance':
        return _plain_balance(s, s['topk_idx'])
    idx, w = _plain_route(s)
    if path == 'route':
        return {'idx': idx, 'weights': w}
    return {'idx': idx, 'weights': w, **_plain_balance(s, idx, s['d_weights'])}


def work(case):
    c = case
    t, size = c['tokens'], {'bf16': 2, 'fp16': 2, 'fp32': 4}
    if c['path'] in ('norm', 'norm grad'):
        h, b, r = c['hidden'], size[c['dtype']], size[c['stream']]
        gate = {'none': 0, 'channel': h, 'token': t, 'element': t * h}[c['gate']] * b
        weights = (c['post'] + c['pre']) * h * b
        if c['path'] == 'norm':
            return {'bytes': t * h * (2 * r + b + b * c['pre']) + gate + weights, 'flops': t * h * (3 + 4 * c['post'] + 4 * c['pre'])}
        # without a norm of the stream, its gradient does not depend on the stream itself, nor that of y on y without norm or gate
        reads = t * h * (r + (b + r) * c['pre'] + b * (c['post'] or c['pre'] or c['gate'] != 'none'))
        return {'bytes': reads + t * h * (r + b) + 2 * gate + 2 * weights, 'flops': t * h * (4 + 12 * c['post'] + 12 * c['pre'])}
    e, k, n = c['experts'], c['topk'], max(1, c['sequences'])
    logits = t * e * size[c['dtype']]
    routes = t * k * 12                                                    # int64 expert and float weight per slot
    losses = n * e * 8
    bytes_ = {'route': logits + routes, 'balance': 2 * logits + t * k * 8 + losses, 'router step': 2 * logits + routes + t * k * 4 + losses}[c['path']]
    return {'bytes': bytes_ + t * (c['padded'] > 0), 'flops': t * e * {'route': 6, 'balance': 20, 'router step': 26}[c['path']]}


# ---------------------------------------------------------------- the definitions in 64 bits; gradients by differentiation

def _exact_norm(c, s):
    grad = c['path'] == 'norm grad'
    x = {k: s[k].double().requires_grad_(grad) for k in ('residual', 'y', 'gate', 'post', 'pre') if s[k] is not None}

    def normed(v, w):
        return v / torch.sqrt(torch.sum(v ** 2, dim=1, keepdim=True) / c['hidden'] + EPS) * (w + c['offset'])
    update = normed(x['y'], x['post']) if c['post'] else x['y']
    stream = x['residual'] + (x['gate'] * update if 'gate' in x else update) * c['scale']
    after = normed(stream, x['pre']) if c['pre'] else None
    if not grad:
        return _given({'stream': stream, 'normed': after})
    loss = (stream * s['d_stream'].double()).sum()
    if c['pre']:
        loss = loss + (after * s['d_normed'].double()).sum()
    loss.backward()
    return {k: v.grad for k, v in x.items()}


def _exact_router(c, s):
    t, e, k = c['tokens'], c['experts'], c['topk']
    l = s['logits'].double().requires_grad_(True)
    out = {}
    if c['path'] == 'balance':
        idx = s['topk_idx']
    else:
        keys = l.detach().cpu().numpy()
        if s['bias'] is not None:
            keys = 1.0 / (1.0 + np.exp(-keys)) + s['bias'].double().cpu().numpy()
        idx = torch.from_numpy(np.argsort(-keys, axis=1, kind='stable')[:, :k].copy()).cuda()
        if s['valid'] is not None:
            idx[~s['valid']] = -1
    on = torch.zeros((t, k, e), dtype=torch.bool, device='cuda') if t * k * e <= 1 << 26 else None
    if on is None:
        hot = torch.zeros((t, e), dtype=torch.float64, device='cuda')
        for j in range(k):
            hot[torch.arange(t, device='cuda'), idx[:, j].clamp(min=0)] += (idx[:, j] >= 0).double()
    else:
        on.scatter_(2, idx.clamp(min=0)[:, :, None], (idx >= 0)[:, :, None])
        hot = on.double().sum(dim=1)
    loss = 0.0
    if c['path'] != 'balance':
        scores = torch.sigmoid(l) if s['bias'] is not None else torch.exp(l - l.amax(dim=1, keepdim=True).detach())
        chosen = torch.where(idx >= 0, scores.gather(1, idx.clamp(min=0)), 0.0)
        w = _route_scale(s) * chosen / chosen.sum(dim=1, keepdim=True).clamp(min=1e-300)
        out['idx'], out['weights'] = idx, w.detach()
        if c['path'] == 'route':
            return out
        loss = loss + (w * s['d_weights'].double()).sum()
    if s['bias'] is None:
        p = torch.softmax(l, dim=1)
    else:
        p = torch.sigmoid(l)
        p = p / p.sum(dim=1, keepdim=True)
    cuts = [0, t] if s['cu_seqlens'] is None else s['cu_seqlens'].tolist()
    routed = (idx >= 0).any(dim=1)
    balance, z, live, everyone, counts, mean, tokens = 0.0, 0.0, 0, 0, [], [], []
    for a, b in zip(cuts[:-1], cuts[1:]):
        rows = torch.arange(a, b, device='cuda')[routed[a:b]]
        n = rows.numel()
        counts.append(hot[rows].sum(dim=0))
        mean.append(p[rows].sum(dim=0) / max(1, n))
        tokens.append(n)
        if n:
            balance = balance + (counts[-1] * mean[-1]).sum() * (e / (k * n))
            z = z + (torch.logsumexp(l[rows], dim=1) ** 2).sum()
            live, everyone = live + 1, everyone + n
    balance, z = balance / max(1, live), z / max(1, everyone)
    total = BALANCE * balance + Z * z
    if everyone or c['path'] == 'router step':
        (loss + s['d_loss'] * total).backward()
    out['losses'] = torch.tensor([float(total), float(balance), float(z)], dtype=torch.float64)
    out['counts'], out['mean_probs'] = torch.stack(counts).int(), torch.stack(mean).detach()
    out['tokens'] = torch.tensor(tokens, dtype=torch.int32)
    out['d_logits'] = l.grad if l.grad is not None else torch.zeros_like(l).detach()
    return out


def exact(case, seed):
    s = prepare(case, seed)
    return _exact_norm(case, s) if case['path'] in ('norm', 'norm grad') else _exact_router(case, s)
