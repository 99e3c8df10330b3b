"""`block_norm` and `block_norm_backward` on the GPU against plain forms in 64 bits (tolerances: util_block)."""
import pytest
import torch

import hopper_megamoe_basedondeepgemm_b200 as mm
from tests import util_block as B

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32
CHAIN = 64                                     # of a stream or normed element: ROW / 2 and 4 for each of two roots, and a dozen products
GRAD_CHAIN = 192                               # of a gradient's element: three of those sums one after the other


def _inputs(tokens, hidden, dtype=BF16, stream=None, weight=None, gate='none', post=True, pre=True, y=True, seed=0, offset=0.0):
    g = torch.Generator(device='cuda').manual_seed(seed)

    def randn(*shape):
        return torch.randn(shape, generator=g, device='cuda')
    x = dict(residual=(randn(tokens, hidden) * torch.exp(0.5 * randn(hidden))).to(stream or dtype), y=randn(tokens, hidden).to(dtype) if y else None)
    x['pre_weight'] = (1.0 - offset + 0.2 * randn(hidden)).to(weight or dtype) if pre else None
    x['post_weight'] = (1.0 - offset + 0.2 * randn(hidden)).to(weight or dtype) if post else None
    shape = {'none': None, 'channel': (hidden,), 'token': (tokens, 1), 'element': (tokens, hidden)}[gate]
    x['gate'] = torch.sigmoid(randn(*shape)).to(dtype) if shape else None
    return x, randn(tokens, hidden).to(stream or dtype), randn(tokens, hidden).to(dtype) if pre else None


def _check_forward(x, out, scale=1.0, eps=1e-6, offset=0.0):
    ref, normed, size, normed_size = B.norm_reference(x['residual'], x['y'], x['pre_weight'], x['post_weight'], x['gate'], scale, eps, offset)
    if x['y'] is not None:
        B.assert_near(out[0], ref, size, CHAIN, 'stream')
    if x['pre_weight'] is not None:
        B.assert_near(out[1], normed, normed_size, CHAIN, 'normed')
    else:
        assert out[1] is None


def _check_gradients(x, d_stream, d_normed, grads, scale=1.0, eps=1e-6, offset=0.0):
    args = (d_stream, d_normed, x['residual'], x['y'], x['pre_weight'], x['post_weight'], x['gate'], scale, eps, offset)
    ref, size = B.norm_gradients(*args), B.norm_gradient_magnitudes(*args)
    tokens, hidden = x['residual'].shape
    for name in ('residual', 'y', 'gate', 'pre_weight', 'post_weight'):
        got = getattr(grads, name)
        assert (got is None) == (name not in ref), name
        if got is None:
            continue
        assert got.dtype == x[name].dtype and got.shape == x[name].shape
        # a weight's gradient: one addition per row of a CTA and per CTA at most
        chain = GRAD_CHAIN + (tokens if name in ('pre_weight', 'post_weight') or got.dim() == 1 else B.ROW)
        B.assert_near(got, ref[name], size[name], chain, name)


SHAPES = [(1, 1), (1, 8), (3, 7), (2, 512), (1, 3072), (5, 1000), (7, 1001), (300, 64), (33, 2048), (4, 4096), (9, 4097), (3, 4104), (2, 8191), (3, 8192), (700, 136)]
KINDS = [dict(), dict(post=False), dict(pre=False), dict(post=False, pre=False), dict(y=False, post=False),
         dict(gate='channel'), dict(gate='token', post=False), dict(gate='element', pre=False), dict(gate='token'), dict(gate='element')]
TYPES = [dict(), dict(stream=FP32), dict(dtype=FP16), dict(dtype=FP16, stream=FP32, weight=FP32), dict(dtype=FP32), dict(weight=FP32)]


@pytest.mark.parametrize('shape', SHAPES)
@pytest.mark.parametrize('types', range(len(TYPES)))
def test_forward_and_gradients(shape, types):
    """Every kind of call at every shape and set of types."""
    for i, kind in enumerate(KINDS):
        offset, scale = (1.0, 0.7) if i % 2 else (0.0, 1.0)
        x, d_stream, d_normed = _inputs(*shape, **TYPES[types], **kind, seed=i, offset=offset)
        if x['y'] is None and x['residual'].dtype != x['pre_weight'].dtype and x['pre_weight'].dtype != FP32:
            normed = torch.empty(shape, dtype=TYPES[types].get('dtype', BF16), device='cuda')
        else:
            normed = None
        if x['y'] is None and normed is None and d_normed is not None:
            d_normed = d_normed.to(x['residual'].dtype)
        out = mm.block_norm(**x, scale=scale, weight_offset=offset, normed=normed)
        _check_forward(x, out, scale, offset=offset)
        grads = mm.block_norm_backward(d_stream, d_normed, **x, scale=scale, weight_offset=offset)
        _check_gradients(x, d_stream, d_normed, grads, scale, offset=offset)


@pytest.mark.parametrize('tokens, hidden', [(2000, 1024), (5000, 100), (1, 8192), (1500, 4096)])
def test_many_rows(tokens, hidden):
    """More rows than the GPU holds at a time, and one."""
    x, d_stream, d_normed = _inputs(tokens, hidden, gate='channel', seed=3)
    _check_forward(x, mm.block_norm(**x))
    grads = mm.block_norm_backward(d_stream, d_normed, **x)
    _check_gradients(x, d_stream, d_normed, grads)
    again = mm.block_norm_backward(d_stream, d_normed, **x)
    assert all(torch.equal(a, b) for a, b in zip(grads, again))            # the same sums in the same order


@pytest.mark.parametrize('hidden', [2056, 2560, 3072])
@pytest.mark.parametrize('tokens', [295, 296, 297, 741])
def test_rows_in_pairs(tokens, hidden):
    """Widths and row counts around those at which a CTA takes two rows at a time, the last pair without its second row."""
    for i, kind in enumerate([dict(), dict(gate='token'), dict(gate='channel', post=False), dict(pre=False), dict(gate='element'), dict(y=False, post=False), dict(gate='token', pre=False)]):
        types = TYPES[(i + tokens) % len(TYPES)]
        x, d_stream, d_normed = _inputs(tokens, hidden, **{**types, 'stream': None}, **kind, seed=i)
        _check_gradients(x, d_stream, d_normed, mm.block_norm_backward(d_stream, d_normed, **x))
        assert all(a is None or torch.equal(a, b) for a, b in zip(mm.block_norm_backward(d_stream, d_normed, **x), mm.block_norm_backward(d_stream, d_normed, **x)))


@pytest.mark.parametrize('hidden', [4097, 4104, 5120, 8190, 8192])
@pytest.mark.parametrize('tokens', [73, 75, 149, 400])
def test_rows_of_two_ctas(tokens, hidden):
    """Rows of more than 4096 channels, around the numbers of pairs of CTAs that a GPU holds: results, and the same ones in every call."""
    for i, kind in enumerate([dict(gate='token'), dict(gate='channel', post=False), dict(pre=False), dict(gate='element'), dict(y=False, post=False), dict()]):
        types = {**TYPES[(i + tokens + hidden) % len(TYPES)], 'stream': None}
        x, d_stream, d_normed = _inputs(tokens, hidden, **types, **kind, seed=i)
        out, grads = mm.block_norm(**x), mm.block_norm_backward(d_stream, d_normed, **x)
        _check_forward(x, out)
        _check_gradients(x, d_stream, d_normed, grads)
        for _ in range(3):                     # one behind the other
            again, grads_again = mm.block_norm(**x), mm.block_norm_backward(d_stream, d_normed, **x)
        assert all(a is None or torch.equal(a, b) for a, b in zip((*out, *grads), (*again, *grads_again)))


def test_one_gradient_only():
    x, d_stream, d_normed = _inputs(40, 512, gate='token')
    grads = mm.block_norm_backward(None, d_normed, **x)
    _check_gradients(x, None, d_normed, grads)
    x, d_stream, _ = _inputs(40, 512, pre=False)
    _check_gradients(x, d_stream, None, mm.block_norm_backward(d_stream, None, **x))
    x, _, d_normed = _inputs(40, 512, y=False, post=False)
    _check_gradients(x, None, d_normed, mm.block_norm_backward(None, d_normed, **x))


@pytest.mark.parametrize('hidden', [256, 250])
def test_no_tokens(hidden):
    x, d_stream, d_normed = _inputs(0, hidden, gate='channel')
    stream, normed = mm.block_norm(**x)
    assert stream.shape == normed.shape == (0, hidden)
    g = mm.block_norm_backward(d_stream, d_normed, **x)
    assert g.residual.shape == g.y.shape == (0, hidden)
    for t in (g.gate, g.pre_weight, g.post_weight):
        assert t.shape == (hidden,) and not t.any()


def test_rows_of_zeros_and_of_extremes():
    """A row without anything in it has a root of eps; infinities and NaN stay in their rows (and in the sums over the rows)."""
    x, d_stream, d_normed = _inputs(6, 512)
    for name in ('residual', 'y'):
        x[name][1] = 0
        x[name][2] = 1e-20
        x[name][3] *= 1e15
    out = mm.block_norm(**x)
    _check_forward(x, out)
    assert not out[0][1].any() and not out[1][1].any()
    _check_gradients(x, d_stream, d_normed, mm.block_norm_backward(d_stream, d_normed, **x))
    x['y'][4, 7], x['residual'][5, 3] = float('inf'), float('nan')
    stream, normed = mm.block_norm(**x)
    assert torch.equal(stream[:4], out[0][:4]) and torch.equal(normed[:4], out[1][:4])
    assert torch.isnan(normed[4:]).all(dim=1).tolist() == [True, True]


@pytest.mark.parametrize('gate', ['none', 'token', 'element', 'channel'])
@pytest.mark.parametrize('hidden, pad', [(512, 8), (512, 3), (96, 0), (131, 1)])
def test_strided_rows(hidden, pad, gate):
    """Rows of a wider buffer, also at odd distances and starts; what lies between them stays as it was."""
    tokens, ld, start = 21, hidden + 2 * pad, pad
    x, d_stream, d_normed = _inputs(tokens, hidden, gate=gate)

    def wide(t):
        buf = torch.full((tokens, ld), 7.0, dtype=t.dtype, device='cuda')
        buf[:, start:start + hidden] = t
        return buf, buf[:, start:start + hidden]
    s = dict(x)
    for name in ('residual', 'y') + (('gate',) if gate == 'element' else ()):
        s[name] = wide(x[name])[1]
    if gate == 'token':
        s['gate'] = torch.stack([x['gate'][:, 0], x['gate'][:, 0] * 0], dim=1)[:, :1]
    (b1, o1), (b2, o2) = wide(torch.zeros_like(x['residual'])), wide(torch.zeros_like(x['y']))
    out = mm.block_norm(**s, residual_out=o1, normed=o2)
    _check_forward(x, out)
    for b in (b1, b2):
        assert bool((b[:, :start] == 7.0).all()) and bool((b[:, start + hidden:] == 7.0).all())
    grads = mm.block_norm_backward(wide(d_stream)[1], wide(d_normed)[1], **s)
    _check_gradients(x, d_stream, d_normed, grads)


@pytest.mark.parametrize('tokens, hidden, pad, start', [(5, 9, 0, 0), (2600, 1001, 0, 0), (2600, 1001, 2, 0), (1300, 2047, 5, 0), (700, 3002, 0, 0), (700, 3002, 1, 1), (400, 4089, 0, 0), (400, 4091, 0, 0),
                                                        (300, 5003, 0, 0), (300, 5003, 4, 3), (160, 8185, 3, 0), (160, 8187, 0, 0), (4000, 67, 0, 0), (4000, 67, 6, 5), (5000, 8, 1, 0), (3000, 5, 0, 0)])
def test_rows_that_start_anywhere(tokens, hidden, pad, start):
    """Rows whose starts lie on no boundary, or the first of which lies on one, more of them than are worked on at a time; NaN between and behind them, which has to stay."""
    ld = hidden + pad

    def among_nan(t):
        if t is None or t.dim() == 1 or t.shape[1] == 1:
            return None, t
        buf = torch.full((start + tokens * ld + 8,), float('nan'), dtype=t.dtype, device='cuda')
        rows = buf[start:start + tokens * ld].view(tokens, ld)[:, :hidden]
        rows.copy_(t)
        return buf, rows
    for i, kind in enumerate([dict(), dict(gate='token', pre=False), dict(gate='element'), dict(y=False, post=False), dict(gate='channel', post=False), dict(gate='token')]):
        types = {**TYPES[(i + tokens + pad) % len(TYPES)]}
        if not kind.get('y', True):
            types['stream'] = None
        x, d_stream, d_normed = _inputs(tokens, hidden, **types, **kind, seed=i)
        s = {name: among_nan(t)[1] for name, t in x.items()}
        bufs = [among_nan(torch.zeros_like(x[name])) if x[name] is not None else (None, None) for name in ('residual', 'y')]
        buf_n, normed = among_nan(torch.zeros_like(d_normed)) if d_normed is not None else (None, None)
        out = mm.block_norm(**s, residual_out=bufs[0][1] if x['y'] is not None else None, normed=normed)
        _check_forward(x, out)
        for buf, rows in ((bufs[0][0] if x['y'] is not None else None, out[0]), (buf_n, out[1])):
            if buf is not None:
                rows.zero_()
                assert int(torch.isnan(buf).sum()) == buf.numel() - tokens * hidden
        grads = mm.block_norm_backward(among_nan(d_stream)[1], among_nan(d_normed)[1], **s)
        _check_gradients(x, d_stream, d_normed, grads)
        again = mm.block_norm_backward(among_nan(d_stream)[1], among_nan(d_normed)[1], **s)
        assert all(a is None or torch.equal(a, b) for a, b in zip(grads, again))
        if x['y'] is not None and pad == 0 and start == 0:       # in place
            stream, y = x['residual'].clone(), x['y'].clone()
            once = mm.block_norm(**x)
            twice = mm.block_norm(**{**x, 'residual': stream, 'y': y}, residual_out=stream, normed=y if x['pre_weight'] is not None else None)
            assert torch.equal(once[0], twice[0]) and (once[1] is None or torch.equal(once[1], twice[1]))


def test_rows_far_apart():
    """Element offsets beyond 32 bits."""
    hidden, ld = 256, 2 ** 31 // 2 + 8
    buf = torch.empty(2 * ld + hidden, dtype=BF16, device='cuda')
    far = torch.as_strided(buf, (3, hidden), (ld, 1))
    x, d_stream, d_normed = _inputs(3, hidden)
    far.copy_(x['y'])
    s = dict(x, y=far)
    _check_forward(x, mm.block_norm(**s))
    _check_gradients(x, d_stream, d_normed, mm.block_norm_backward(d_stream, d_normed, **s))
    out = mm.block_norm(**s, normed=far)[1]                                 # in place, too
    assert out.data_ptr() == far.data_ptr()
    _check_forward(x, (mm.block_norm(**x)[0], far))


@pytest.mark.parametrize('hidden', [512, 77])
@pytest.mark.parametrize('tokens', [1, 900])
def test_in_place(tokens, hidden):
    x, _, _ = _inputs(tokens, hidden)
    want = mm.block_norm(**x)
    s = {k: v.clone() if v is not None else None for k, v in x.items()}
    got = mm.block_norm(**s, residual_out=s['residual'], normed=s['y'])
    assert got[0] is s['residual'] and got[1] is s['y']
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    r = x['residual'].clone()                                               # the next block's input over the old stream, the new one elsewhere
    got = mm.block_norm(r, x['y'], pre_weight=x['pre_weight'], post_weight=x['post_weight'], normed=r)
    assert torch.equal(got[0], want[0]) and torch.equal(r, want[1])


def test_writes_are_known_to_autograd():
    """A tensor that something has saved for its backward pass and that is then written in place is refused there, as torch's own operators have it."""
    x, _, _ = _inputs(8, 64, dtype=FP32)
    w = torch.ones(8, 64, device='cuda', requires_grad=True)
    product = w * x['residual']                                             # saves the stream
    mm.block_norm(x['residual'], x['y'], pre_weight=x['pre_weight'], residual_out=x['residual'])
    with pytest.raises(RuntimeError):
        product.sum().backward()
    with torch.inference_mode():
        r = x['y'].clone()
        mm.block_norm(r, x['y'], pre_weight=x['pre_weight'], residual_out=r)


def test_captured_and_replayed():
    """A graph of both directions, replayed with new inputs, beside another graph of the same calls."""
    x, d_stream, d_normed = _inputs(300, 1024, gate='channel')
    mm.block_norm(**x), mm.block_norm_backward(d_stream, d_normed, **x)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = mm.block_norm(**x)
            grads = mm.block_norm_backward(d_stream, d_normed, **x)
        graphs.append((g, out, grads))
    new, new_ds, new_dn = _inputs(300, 1024, gate='channel', seed=9)
    for k in x:
        x[k].copy_(new[k])
    d_stream.copy_(new_ds), d_normed.copy_(new_dn)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for s, (g, _, _) in zip(streams, graphs):
        with torch.cuda.stream(s):
            g.replay()
    torch.cuda.synchronize()
    want, want_grads = mm.block_norm(**new), mm.block_norm_backward(new_ds, new_dn, **new)
    for _, out, grads in graphs:
        assert all(torch.equal(a, b) for a, b in zip(out, want)) and all(torch.equal(a, b) for a, b in zip(grads, want_grads))


def test_two_streams_at_once():
    sets = [_inputs(2500, 1024, gate='channel', seed=s) for s in range(2)]
    want = [mm.block_norm_backward(ds, dn, **x) for x, ds, dn in sets]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                x, ds, dn = sets[i]
                got[i].append(mm.block_norm_backward(ds, dn, **x))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(a, b) for g in got[i] for a, b in zip(g, want[i]))


def test_against_differences():
    """The gradient of a scalar of the outputs against its differences along random directions, 32-bit inputs: a step of 2^-6 leaves an error of its
    square times the third derivative, under 2 % of the gradient here; the sums' roundings are far below that."""
    x, ds, dn = _inputs(16, 256, dtype=FP32, gate='element', seed=4)
    grads = mm.block_norm_backward(ds, dn, **x, scale=0.8)

    def value(**change):
        stream, normed = mm.block_norm(**{**x, **change}, scale=0.8)
        return float((stream.double() * ds.double()).sum() + (normed.double() * dn.double()).sum())
    for name in ('residual', 'y', 'gate', 'pre_weight', 'post_weight'):
        way = getattr(grads, name)                                           # along the gradient itself the slope is its square
        way = way / way.norm()
        step = 2.0 ** -6
        slope = (value(**{name: x[name] + step * way}) - value(**{name: x[name] - step * way})) / (2 * step)
        want = float((getattr(grads, name).double() * way.double()).sum())
        assert abs(slope - want) <= 0.02 * abs(want), name


def test_refusals():
    x, ds, dn = _inputs(8, 64)
    r, y, w = x['residual'], x['y'], x['pre_weight']
    bad = [
        lambda: mm.block_norm(r[0], y, pre_weight=w), lambda: mm.block_norm(r, y[:7], pre_weight=w), lambda: mm.block_norm(r, y.half(), pre_weight=w),
        lambda: mm.block_norm(r, y.float(), pre_weight=w), lambda: mm.block_norm(r.double(), y, pre_weight=w), lambda: mm.block_norm(r, y.cpu(), pre_weight=w),
        lambda: mm.block_norm(r.t(), y.t(), pre_weight=w[:8]), lambda: mm.block_norm(r, y, pre_weight=w[:63]), lambda: mm.block_norm(r, y, pre_weight=w.half()),
        lambda: mm.block_norm(r, y, pre_weight=w, post_weight=w.float()), lambda: mm.block_norm(r, y, pre_weight=w[::2]), lambda: mm.block_norm(r, y, pre_weight=w.cpu()),
        lambda: mm.block_norm(r, y, pre_weight=w, gate=r[:, :2]), lambda: mm.block_norm(r, y, pre_weight=w, gate=r[:7]), lambda: mm.block_norm(r, y, gate=r[:, 0]),
        lambda: mm.block_norm(r, y, gate=w.half()), lambda: mm.block_norm(r), lambda: mm.block_norm(r, pre_weight=w, gate=w), lambda: mm.block_norm(r, pre_weight=w, post_weight=w),
        lambda: mm.block_norm(r, pre_weight=w, residual_out=r), lambda: mm.block_norm(r, y, normed=y), lambda: mm.block_norm(r, y, pre_weight=w, eps=0.0),
        lambda: mm.block_norm(r, y, pre_weight=w, scale=float('nan')), lambda: mm.block_norm(r, y, pre_weight=w, residual_out=y, normed=y),
        lambda: mm.block_norm(r, y, pre_weight=w, residual_out=r[:7]), lambda: mm.block_norm(r, y, pre_weight=w, normed=y.float()),
        lambda: mm.block_norm(r[:4], y[:4], residual_out=r[1:5]), lambda: mm.block_norm(r, y, residual_out=r[:1].expand(8, 64)),
        lambda: mm.block_norm(torch.zeros(1, 8200, device='cuda'), pre_weight=torch.ones(8200, device='cuda')),
        lambda: mm.block_norm_backward(ds, None, r, y, pre_weight=w), lambda: mm.block_norm_backward(ds, dn, r, y), lambda: mm.block_norm_backward(None, None, r, y),
        lambda: mm.block_norm_backward(ds[:7], dn, r, y, pre_weight=w), lambda: mm.block_norm_backward(ds.float(), dn, r, y, pre_weight=w),
        lambda: mm.block_norm_backward(ds, dn.float(), r, y, pre_weight=w), lambda: mm.block_norm_backward(ds, dn, r, y, pre_weight=w, eps=-1.0),
    ]
    for i, f in enumerate(bad):
        with pytest.raises(RuntimeError):
            f()
            print('not refused:', i)
