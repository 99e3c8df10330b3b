"""Plain forms in 64 bits of the operators around the layer, and how far a result may be from them.

Tolerances count roundings. An output is rounded once to its type, half a step: `eps / 2` of its value (plus half the smallest subnormal number of
fp16). Before that everything is 32-bit arithmetic; with u = 2^-24, a result that is a sum of terms is off by at most a number of u times the sum
of the terms' magnitudes, where the number counts the roundings that a term passes through: a handful of products, the roots and exponentials
(two units in the last place, so 4 u), and a sum's longest chain of additions.
"""
import torch

U = 2.0 ** -24


def rounding(ref, dtype):
    tiny = {torch.float16: 2.0 ** -25}.get(dtype, 0.0)
    return ref.abs() * (torch.finfo(dtype).eps / 2) + tiny


def assert_near(got, ref, magnitude, chain, what):
    """|got - ref| <= rounding to got's type + chain * u * magnitude, element by element."""
    assert got.shape == ref.shape, what
    ref, magnitude = ref.detach(), magnitude.detach()
    off = (got.double() - ref).abs()
    # (the rounding is that of the computed value, which is off from the reference's by the second part: hence the factor)
    limit = (rounding(ref, got.dtype) + chain * U * magnitude) * (1 + torch.finfo(got.dtype).eps)
    bad = ~(off <= limit)
    assert not bool(bad.any()), f'{what}: {int(bad.sum())} of {bad.numel()}, worst {float((off / limit.clamp(min=1e-300)).max()):.2f} of the limit'


# A row's sum of squares: 16 elements one after the other in a thread at most, 5 steps over a warp, 16 warps; halved by the root, which adds 4 u.
ROW = 16 + 5 + 16


def norm_reference(residual, y, pre, post, gate, scale, eps, offset):
    """(stream, normed, and the sums of magnitudes that their errors go by), all in 64 bits."""
    r = residual.double()
    v, size_v = torch.zeros_like(r), torch.zeros_like(r)
    if y is not None:
        u = y.double()
        if post is not None:
            u = u / torch.sqrt((u ** 2).mean(dim=1, keepdim=True) + eps) * (post.double() + offset)
        v = u * scale if gate is None else u * gate.double() * scale
        size_v = v.abs()
        if post is not None and offset != 0.0:           # offset + w is rounded: it counts as much as it would without cancelling
            size_v = size_v * ((post.double().abs() + abs(offset)) / (post.double() + offset).abs().clamp(min=1e-30))
    stream = r + v
    size = r.abs() + size_v
    if pre is None:
        return stream, None, size, None
    inv = 1.0 / torch.sqrt((stream ** 2).mean(dim=1, keepdim=True) + eps)
    w = pre.double() + offset
    normed = stream * inv * w
    # the root's own error goes by how much of the stream's squares its terms' errors make up
    spread = (stream.abs() * size).mean(dim=1, keepdim=True) * inv ** 2
    return stream, normed, size, (size * inv + stream.abs() * inv * (1 + spread)) * (pre.double().abs() + abs(offset))


def norm_gradients(d_stream, d_normed, residual, y, pre, post, gate, scale, eps, offset):
    """Gradients by differentiation in 64 bits: {name: tensor}."""
    x = {k: t.double().requires_grad_(True) for k, t in (('residual', residual), ('y', y), ('gate', gate), ('pre_weight', pre), ('post_weight', post)) if t is not None}
    stream, normed, _, _ = norm_reference(x['residual'], x.get('y'), x.get('pre_weight'), x.get('post_weight'), x.get('gate'), scale, eps, offset)
    loss = 0.0
    if d_stream is not None:
        loss = loss + (stream * d_stream.double()).sum()
    if d_normed is not None:
        loss = loss + (normed * d_normed.double()).sum()
    loss.backward()
    return {k: v.grad if v.grad is not None else torch.zeros_like(v) for k, v in x.items()}


def norm_gradient_magnitudes(d_stream, d_normed, residual, y, pre, post, gate, scale, eps, offset):
    """The gradients with every term's magnitude in place of the term: what their errors go by."""
    r = residual.double().abs()
    one = torch.ones(1, dtype=torch.float64, device=r.device)
    g = gate.double().abs() if gate is not None else one
    w1 = post.double().abs() + abs(offset) if post is not None else one
    out = {}
    n1 = i1 = None
    if y is not None:
        a = y.double().abs()
        i1 = 1.0 / torch.sqrt((a ** 2).mean(dim=1, keepdim=True) + eps) if post is not None else one
        n1 = a * i1
    d = d_stream.double().abs() if d_stream is not None else torch.zeros_like(r)
    if d_normed is not None:
        exact = norm_reference(residual, y, None, post, gate, scale, eps, offset)[0]
        size = r + (abs(scale) * g * n1 * w1 if y is not None else 0.0)
        i2 = 1.0 / torch.sqrt((exact ** 2).mean(dim=1, keepdim=True) + eps)
        n2 = size * i2
        n2 = n2 * (1 + (n2 ** 2).mean(dim=1, keepdim=True))                 # (and what the error of the root adds)
        dn = d_normed.double().abs() * (pre.double().abs() + abs(offset))
        d = d + i2 * (dn + n2 * (dn * n2).mean(dim=1, keepdim=True)) * (1 + (n2 ** 2).mean(dim=1, keepdim=True))
        out['pre_weight'] = (d_normed.double().abs() * n2).sum(dim=0)
    out['residual'] = d
    if y is None:
        return out
    dv = abs(scale) * d
    dg = dv * n1 * w1
    if gate is not None:
        out['gate'] = dg if gate.shape == r.shape else (dg.sum(dim=1, keepdim=True) if gate.dim() == 2 else dg.sum(dim=0))
        if gate.shape == r.shape and gate.dim() == 2:
            out['gate'] = dg
    du = dv * g
    out['y'] = du
    if post is not None:
        out['post_weight'] = (du * n1).sum(dim=0)
        dn1 = du * w1
        out['y'] = i1 * (dn1 + n1 * (dn1 * n1).mean(dim=1, keepdim=True))
    return out


def route_reference(logits, topk, mode, bias, valid, scale):
    """(idx, weights in 64 bits) by sorting in numpy, where equal keys keep their order."""
    import numpy as np
    l = logits.double().cpu().numpy()
    off = ~(l > -np.inf)
    with np.errstate(all='ignore'):
        key = l if mode == 0 else 1.0 / (1.0 + np.exp(-l)) + (bias.double().cpu().numpy() if bias is not None else 0.0)
    key = np.where(off, -np.inf, key)
    order = np.argsort(-key, axis=1, kind='stable')[:, :topk]
    live = np.take_along_axis(~off, order, 1)
    if valid is not None:
        live &= (valid.cpu().numpy() != 0)[:, None]
    idx = np.where(live, order, -1)
    return torch.from_numpy(idx).to(logits.device), route_weights(logits, torch.from_numpy(idx).to(logits.device), mode, scale).detach()


def clean_logits(logits):
    """64-bit logits as they count: NaN is an expert that is off, +inf the largest 32-bit number."""
    l = logits.double()
    l = torch.where(torch.isnan(l.detach()), torch.full_like(l, -float('inf')), l)
    return l.clamp(max=torch.finfo(torch.float32).max)


def route_weights(logits, idx, mode, scale):
    """The weights of given routes, differentiable in 64-bit logits; 0 where there is no route."""
    l = clean_logits(logits)
    live = (idx >= 0) & (idx < logits.shape[1])
    chosen = l.gather(1, torch.where(live, idx, 0))
    live = live & (chosen.detach() > -float('inf'))
    if mode == 0:
        top = torch.where(live, chosen.detach(), -float('inf')).amax(dim=1, keepdim=True)
        s = torch.exp(torch.where(live, chosen - torch.where(top > -float('inf'), top, 0.0), 0.0))
    else:
        s = torch.sigmoid(torch.where(live, chosen, 0.0))
    s = torch.where(live, s, 0.0)
    total = s.sum(dim=1, keepdim=True)
    return s / torch.where(total > 0, total, 1.0) * scale


def balance_reference(logits, idx, mode, cu, balance_coef, z_coef):
    """losses [3], counts, mean_probs, tokens of 64-bit logits that may ask for a gradient. Experts that are off take no part."""
    t, e = logits.shape
    k = idx.shape[1]
    l = clean_logits(logits)
    on = l.detach() > -float('inf')
    any_on = on.any(dim=1, keepdim=True)
    safe = torch.where(on, l, 0.0)
    top = torch.where(on, safe.detach(), -float('inf')).amax(dim=1, keepdim=True)
    top = torch.where(any_on, top, 0.0)
    ex = torch.where(on, torch.exp(torch.where(on, safe - top, 0.0)), 0.0)
    total = ex.sum(dim=1, keepdim=True)
    lse = torch.where(any_on, top + torch.log(torch.where(any_on, total, 1.0)), 0.0)[:, 0]
    if mode == 1:
        ex = torch.where(on, torch.sigmoid(safe), 0.0)
        total = ex.sum(dim=1, keepdim=True)
    p = ex / torch.where(total > 0, total, 1.0)
    live = (idx >= 0) & (idx < e)
    hot = torch.zeros((t, e), dtype=torch.float64, device=logits.device)
    hot.scatter_add_(1, torch.where(live, idx, 0), live.double())
    routed = live.any(dim=1)
    cuts = [0, t] if cu is None else cu.tolist()
    counts, mean, tokens, balance, z = [], [], [], 0.0, 0.0
    for a, b in zip(cuts[:-1], cuts[1:]):
        rows = torch.arange(a, b, device=logits.device)[routed[a:b]]
        n = rows.numel()
        counts.append(hot[rows].sum(dim=0))
        mean.append(p[rows].sum(dim=0) / max(n, 1))
        tokens.append(n)
        if n:
            balance = balance + (counts[-1] * mean[-1]).sum() * e / (k * n)
            z = z + (lse[rows] ** 2).sum()
    balance, z = balance / max(1, sum(n > 0 for n in tokens)), z / max(1, sum(tokens))
    total = balance_coef * balance + z_coef * z
    losses = [v if isinstance(v, torch.Tensor) else torch.zeros((), dtype=torch.float64, device=logits.device) for v in (total, balance, z)]
    return torch.stack(losses), torch.stack(counts).int(), torch.stack(mean), torch.tensor(tokens, dtype=torch.int32, device=logits.device)
