"""Attention over an encoder's states against the formula in 64 bits."""
import math

import pytest
import torch

import mxnet_amd as mx
from mxnet_amd import autograd

DEVICES = ['cpu', pytest.param('cuda:0', marks=pytest.mark.gpu)]
TYPES = [torch.float16, torch.bfloat16, torch.float32]
U32 = 2.0 ** -24
nd = mx.nd.from_torch

# batch, heads, shared heads, queries, keys, head size
SIZES = [(1, 1, 1, 1, 1, 8), (2, 3, 1, 5, 7, 16), (1, 2, 2, 3, 9, 5),
         (2, 4, 2, 1, 63, 64), (1, 2, 1, 33, 65, 40), (2, 4, 2, 64, 64, 64),
         (1, 2, 2, 130, 200, 64), (2, 1, 1, 32, 1, 128),
         (3, 12, 4, 77, 129, 64), (1, 8, 2, 1, 1000, 128),
         (2, 2, 2, 1, 4097, 80), (1, 2, 1, 300, 70, 128),
         (1, 4, 1, 16, 1030, 33), (1, 1, 1, 2, 8200, 64),
         (1, 1, 1, 2050, 33, 32)]


def make(size, dtype, device, layout='NTC', seed=0, apart=False, lengths=None,
         mask=False):
    B, H, Hk, sq, sk, D = size
    g = torch.Generator().manual_seed(seed)

    def r(n, width):
        shape = (B, n, width) if layout == 'NTC' else (n, B, width)
        return torch.randn(*shape, generator=g).to(dtype).to(device)

    d = dict(q=r(sq, H * D), dout=r(sq, H * D), values=None, length=None,
             mask=None)
    if apart:
        d['kv'], d['values'] = r(sk, Hk * D), r(sk, Hk * D)
    else:
        d['kv'] = r(sk, 2 * Hk * D)
    if lengths is not None:
        d['length'] = torch.tensor(lengths, device=device)
    if mask:
        d['mask'] = (torch.rand(B, sk, generator=g) < 0.6).to(device)
    return d


def kept(d, size):
    B, sk = size[0], size[4]
    keep = torch.ones(B, sk, dtype=torch.bool, device=d['q'].device)
    if d['length'] is not None:
        keep &= torch.arange(sk, device=keep.device) < d['length'][:, None]
    if d['mask'] is not None:
        keep &= d['mask'].bool()
    return keep


def oracle(d, size, layout):
    """Exact results, and how far rounding may take a kernel from them."""
    B, H, Hk, sq, sk, D = size
    dtype = d['q'].dtype
    f = torch.finfo(dtype)
    # numbers below float32's normal ones may be taken as zeros on the way
    u = f.eps / 2
    tiny = max(f.smallest_normal * u, torch.finfo(torch.float32).tiny)

    def first(t, n, w):  # [B, n, S, w]
        t = t.double() if layout == 'NTC' else t.double().transpose(0, 1)
        return t.reshape(B, -1, n, w).transpose(1, 2)

    def last(t):
        t = t.transpose(1, 2).reshape(B, t.shape[2], -1)
        return t if layout == 'NTC' else t.transpose(0, 1)

    keep = kept(d, size)[:, None, :, None]
    if d['values'] is None:
        kv = first(d['kv'], Hk, 2 * D)
        k, v = kv[..., :D], kv[..., D:]
    else:
        k, v = first(d['kv'], Hk, D), first(d['values'], Hk, D)
    k = torch.where(keep, k, 0.0).repeat_interleave(H // Hk, 1)
    v = torch.where(keep, v, 0.0).repeat_interleave(H // Hk, 1)
    q, do = first(d['q'], H, D), first(d['dout'], H, D)
    c = 1 / math.sqrt(D)
    s = (q @ k.transpose(-1, -2) * c).masked_fill(
        ~keep.transpose(-1, -2), -math.inf)
    some = keep.any(2, keepdim=True)
    p = torch.where(some, torch.softmax(torch.where(some, s, 0.0), -1), 0.0)
    o = p @ v
    ka, va, qa, ga = k.abs(), v.abs(), q.abs(), do.abs()
    # a score is a sum of D products in 32 bits; the exponential and the sum
    # of the weights add a few steps.  Every weight is within e of its own
    # size, then rounded to the type (tiny: below the normal numbers, where
    # weights are relative to one that is at least 1)
    ds = (D + 4) * U32 * c * (qa @ ka.transpose(-1, -2)).amax(-1, keepdim=True)
    top = torch.where(some, s, 0.0).masked_fill(
        ~keep.transpose(-1, -2), -math.inf).amax(-1, keepdim=True).abs()
    top = torch.where(some, top, 0.0)
    e = 2 * ds + 4 * U32 * top + (64 + sk) * U32
    pv = p @ va
    o_off = pv * (u + e) + tiny * va.sum(2, keepdim=True)
    dv = p.transpose(-1, -2) @ do
    dv_off = p.transpose(-1, -2) @ (ga * (u + e + sq * H * U32)) \
        + tiny * ga.sum(2, keepdim=True)
    dp = do @ v.transpose(-1, -2)
    delta = (do * o).sum(-1, keepdim=True)
    w = p * (dp - delta)
    # the row's dO . O comes from the output as it was stored
    w_off = w.abs() * (u + e) + p * (
        (D + 4) * U32 * (ga @ va.transpose(-1, -2))
        + (ga * (o_off + u * o.abs() + D * U32 * o.abs())).sum(
            -1, keepdim=True)) + tiny * (1 + dp.abs() + delta.abs())
    w_off = w_off * keep.transpose(-1, -2)
    n = sk * U32
    dq, dq_off = w @ k * c, ((w_off + n * w.abs()) @ ka) * c
    n = sq * H * U32
    dk = w.transpose(-1, -2) @ q * c
    dk_off = (w_off + n * w.abs()).transpose(-1, -2) @ qa * c

    def shared(t):
        return t.reshape(B, Hk, -1, sk, D).sum(2)

    dk, dk_off, dv, dv_off = (shared(t) for t in (dk, dk_off, dv, dv_off))
    if d['values'] is None:
        pairs = [(torch.cat([dk, dv], -1), torch.cat([dk_off, dv_off], -1))]
    else:
        pairs = [(dk, dk_off), (dv, dv_off)]
    # each result is rounded to the type at the end
    return [(last(a), last(b * (1 + u) + a.abs() * u * 1.01 + tiny))
            for a, b in [(o, o_off), (dq, dq_off)] + pairs]


def call(d, size, layout, grad=False):
    B, H, Hk = size[:3]
    ins = [d['q'], d['kv']] + ([d['values']] if d['values'] is not None
                               else [])
    ins = [nd(t.detach().requires_grad_(grad)) for t in ins]
    kw = dict(heads=H, kv_heads=Hk, layout=layout,
              valid_length=None if d['length'] is None else nd(d['length']),
              mask=None if d['mask'] is None else nd(d['mask']))
    if not grad:
        return [mx.nd.contrib.encdec_attention(*ins, **kw).to_torch()]
    with autograd.record():
        out = mx.nd.contrib.encdec_attention(*ins, **kw)
    grads = autograd.grad([out], ins, [nd(d['dout'])])
    return [out.to_torch().detach()] + [g.to_torch() for g in grads]


def check(got, want):
    for name, g, (w, off) in zip(['out', 'dq', 'dkv', 'dvalues'], got, want):
        bad = (g.double() - w).abs() > off
        assert g.shape == w.shape and not bad.any(), (
            name, int(bad.sum()), bad.numel(),
            float((g.double() - w).abs().max()),
            float(((g.double() - w).abs() / off).max()))


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('size', SIZES)
def test_against_formula(size, dtype, device):
    """Forward and gradients, ragged lengths (one of zero where there are
    several sequences), with and without a mask."""
    B, sk = size[0], size[4]
    lengths = [sk - sk // 3] + [0] * (B > 1) + [sk + 5] * (B > 2)
    for mask in (False, True):
        d = make(size, dtype, device, lengths=lengths, mask=mask)
        want = oracle(d, size, 'NTC')
        check(call(d, size, 'NTC', grad=True), want)
        check(call(d, size, 'NTC'), want)


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('apart', [False, True])
@pytest.mark.parametrize('layout', ['NTC', 'TNC'])
def test_layouts(layout, apart, dtype, device):
    size = (2, 6, 3, 37, 100, 64)
    d = make(size, dtype, device, layout, seed=1, apart=apart)
    check(call(d, size, layout, grad=True), oracle(d, size, layout))


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('sq', [1, 40, 100])
def test_masked_memory_is_never_read(sq, dtype, device):
    """NaN, infinities and the type's lowest value behind the length and
    under the mask change nothing; their gradients are zeros."""
    size = (3, 4, 2, sq, 90, 64)
    B, _, Hk, _, sk, D = size
    d = make(size, dtype, device, seed=2, lengths=[50, 0, 90], mask=True)
    d['mask'][2, 64:] = False
    want = call(d, size, 'NTC', grad=True)
    drop = ~kept(d, size)
    for bad in (math.nan, math.inf, torch.finfo(dtype).min):
        e = dict(d, kv=d['kv'].masked_fill(drop[:, :, None], bad))
        got = call(e, size, 'NTC', grad=True)
        for g, w in zip(got, want):
            assert torch.equal(g, w)
        assert not got[2][drop].any()
    assert not want[0][1].any() and not want[1][1].any()


@pytest.mark.parametrize('device', DEVICES)
def test_large_scores(device):
    """Scores far apart: the running maximum moves by more than exp can
    hold, in both directions along the keys."""
    for flip in (False, True):
        size = (1, 1, 1, 40, 300, 16)
        d = make(size, torch.float32, device, seed=3)
        ramp = torch.linspace(-300, 300, 300, device=device)
        d['kv'][0, :, 0] = ramp.flip(0) if flip else ramp
        d['q'][0, :, 0] = 4.0
        check(call(d, size, 'NTC', grad=True), oracle(d, size, 'NTC'))


def test_gradient_against_differences():
    size = (1, 4, 2, 3, 5, 4)
    d = make(size, torch.float32, 'cpu', seed=4, lengths=[4])
    got = call(d, size, 'NTC', grad=True)

    def value(name, at, step):
        e = dict(d)
        e[name] = d[name].double()
        e[name][at] += step
        o = oracle(e, size, 'NTC')[0][0]
        return float((o * d['dout'].double()).sum())

    for name, g in (('q', got[1]), ('kv', got[2])):
        for at in [(0, 0, 0), (0, 2, 7), (0, 1, 13), (0, 2, 15)]:
            # a smooth function of order one: the difference is off by the
            # square of its step, the gradient by some half steps of float32
            want = (value(name, at, 1e-5) - value(name, at, -1e-5)) / 2e-5
            assert abs(float(g[at]) - want) < 1e-4


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('size', [(2, 2, 1, 0, 5, 8), (2, 2, 1, 3, 0, 8),
                                  (0, 2, 1, 3, 5, 8)])
def test_nothing_to_do(size, device):
    d = make(size, torch.float32, device)
    out, dq, dkv = call(d, size, 'NTC', grad=True)
    assert out.shape == d['q'].shape and dkv.shape == d['kv'].shape
    assert not out.any() and not dq.any() and not dkv.any()


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('sq', [1, 70])
def test_views_on_the_gpu(sq, dtype):
    """Strided inputs, and memory that does not start at 16 bytes."""
    size = (2, 4, 2, sq, 100, 64)
    d = make(size, dtype, 'cuda:0', seed=5)
    want = oracle(d, size, 'NTC')
    wide = torch.randn(2, sq, 300, device='cuda:0').to(dtype)
    wide[:, :, 3:259] = d['q']
    e = dict(d, q=wide[:, :, 3:259])
    check(call(e, size, 'NTC', grad=True), want)
    flat = torch.empty(d['kv'].numel() + 1, device='cuda:0', dtype=dtype)
    flat[1:].copy_(d['kv'].reshape(-1))
    e = dict(d, kv=flat[1:].view(d['kv'].shape))
    check(call(e, size, 'NTC', grad=True), want)


@pytest.mark.gpu
@pytest.mark.parametrize('size', [(2, 4, 2, 1, 3000, 64), (2, 4, 4, 40, 90, 64)])
def test_streams_graphs_and_repeats(size):
    d = make(size, torch.float16, 'cuda:0', seed=6,
             lengths=[size[4], size[4] // 2])
    want = call(d, size, 'NTC', grad=True)
    for _ in range(3):  # no order of sums depends on the schedule
        for a, b in zip(call(d, size, 'NTC', grad=True), want):
            assert torch.equal(a, b)
    sides = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for s in sides:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            outs.append(call(d, size, 'NTC')[0])
    torch.cuda.synchronize()
    for o in outs:
        assert torch.equal(o, want[0])
    # two graphs, replayed in turn: neither uses the other's workspace
    graphs, caught = [], []
    d['length'] = d['length'].to(torch.int32)
    inputs = [dict(d, q=d['q'].clone()), dict(d, q=d['q'].clone())]
    for e in inputs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            caught.append(call(e, size, 'NTC')[0])
        graphs.append(g)
    for k in range(3):
        for e in inputs:
            e['q'].normal_()
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for e, o in zip(inputs, caught):
            assert torch.equal(o, call(e, size, 'NTC')[0])


def test_refusals():
    q, kv = torch.randn(2, 3, 8), torch.randn(2, 5, 8)
    f = mx.nd.contrib.encdec_attention

    def refuse(error, *args, **kw):
        with pytest.raises(error):
            f(*[nd(a) for a in args],
              **{k: nd(v) if isinstance(v, torch.Tensor) else v
                 for k, v in kw.items()})

    f(nd(q), nd(kv), heads=2, kv_heads=1)
    refuse(TypeError, q.double(), kv.double(), heads=2, kv_heads=1)
    refuse(TypeError, q, kv.half(), heads=2, kv_heads=1)
    refuse(ValueError, q, kv, heads=2, kv_heads=2)
    refuse(ValueError, q, kv, heads=3, kv_heads=1)
    refuse(ValueError, q, kv, heads=2, kv_heads=0)
    refuse(ValueError, q, kv, heads=0)
    refuse(ValueError, q[0], kv, heads=2, kv_heads=1)
    refuse(ValueError, q, kv[:1], heads=2, kv_heads=1)
    refuse(ValueError, q, kv, kv[:, :4], heads=1)
    refuse(ValueError, q, kv, heads=2, kv_heads=1, layout='CNT')
    refuse(ValueError, q, kv, heads=2, kv_heads=1,
           valid_length=torch.tensor([1]))
    refuse(ValueError, q, kv, heads=2, kv_heads=1,
           valid_length=torch.tensor([1.0, 2.0]))
    refuse(ValueError, q, kv, heads=2, kv_heads=1,
           mask=torch.ones(2, 4, dtype=torch.bool))
    refuse(ValueError, q, kv, heads=2, kv_heads=1, mask=torch.ones(2, 5))


@pytest.mark.gpu
def test_refusals_on_the_gpu():
    q = torch.randn(1, 2, 136, device='cuda:0')
    with pytest.raises(ValueError):
        mx.nd.contrib.encdec_attention(nd(q), nd(q), nd(q), heads=1)
    with pytest.raises(ValueError):
        mx.nd.contrib.encdec_attention(nd(q), nd(q.cpu()), nd(q), heads=2)


@pytest.mark.parametrize('device', DEVICES)
def test_lengths_that_int32_does_not_hold(device):
    size = (3, 2, 1, 2, 9, 8)
    far = [(1 << 32) + 2, -(1 << 40), 1 << 31]
    d = make(size, torch.float32, device, seed=8, lengths=far)
    check(call(d, size, 'NTC', grad=True), oracle(d, size, 'NTC'))


@pytest.mark.gpu
@pytest.mark.parametrize('sq', [1, 40])
@pytest.mark.parametrize('layout', ['NTC', 'TNC'])
def test_keys_past_2_31_elements(layout, sq):
    """Keys of 4 GB, of which the mask leaves the first ten and the last
    seventy, give what those eighty alone give."""
    sk = (1 << 21) + 100
    few, many = (1, 8, 8, sq, 80, 64), (1, 8, 8, sq, sk, 64)
    d = make(few, torch.bfloat16, 'cuda:0', layout, seed=9)
    shape = list(d['kv'].shape)
    time = 1 if layout == 'NTC' else 0
    shape[time] = sk
    e = dict(d, kv=torch.full(shape, math.nan, dtype=torch.bfloat16,
                              device='cuda:0'),
             mask=torch.zeros(1, sk, dtype=torch.bool, device='cuda:0'))
    for at, to, n in ((0, 0, 10), (10, sk - 70, 70)):
        e['kv'].narrow(time, to, n).copy_(d['kv'].narrow(time, at, n))
        e['mask'][:, to:to + n] = True
    got = call(e, many, layout, grad=True)
    rest = got[2].narrow(time, 10, sk - 80)
    assert not rest.any()
    got[2] = torch.cat([got[2].narrow(time, 0, 10),
                        got[2].narrow(time, sk - 70, 70)], time)
    check(got, oracle(d, few, layout))


@pytest.mark.gpu
@pytest.mark.parametrize('size', [(2, 4, 2, 1, 3000, 64), (2, 4, 4, 40, 90, 64)])
def test_captured_backward(size):
    """Forward and backward in one graph, replayed with eager work between."""
    d = make(size, torch.bfloat16, 'cuda:0', seed=10,
             lengths=[size[4], size[4] // 2])
    d['length'] = d['length'].to(torch.int32)
    call(d, size, 'NTC', grad=True)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        caught = call(d, size, 'NTC', grad=True)
    for k in range(3):
        e = make(size, torch.bfloat16, 'cuda:0', seed=20 + k)
        for name in ('q', 'kv', 'dout'):
            with torch.no_grad():
                d[name].copy_(e[name])
        g.replay()
        torch.cuda.synchronize()
        for a, b in zip(caught, call(d, size, 'NTC', grad=True)):
            assert torch.equal(a, b)


@pytest.mark.gpu
def test_more_refusals_on_the_gpu():
    def zeros(*shape):
        return nd(torch.zeros(*shape, dtype=torch.float16, device='cuda:0'))
    f = mx.nd.contrib.encdec_attention
    many = 1 << 24  # sequences: 2^32 threads
    with pytest.raises(RuntimeError):
        f(zeros(many, 1, 1), zeros(many, 1, 2))
    heads = (1 << 20) + 1
    with pytest.raises(RuntimeError):
        f(zeros(1, 1, heads), zeros(1, 1, 2), heads=heads, kv_heads=1)
    q = torch.randn(1, 2, 8, device='cuda:0', requires_grad=True)
    kv = nd(torch.randn(1, 3, 16, device='cuda:0'))
    with autograd.record():
        o = f(nd(q), kv)
    dq, = autograd.grad([o], [nd(q)], create_graph=True, retain_graph=True)
    with pytest.raises(RuntimeError):  # no second derivatives
        dq.to_torch().square().sum().backward()


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('size', [(2, 4, 2, 40, 100, 96), (1, 2, 1, 1, 700, 72),
                                  (1, 3, 3, 200, 65, 80), (1, 4, 2, 9, 3000, 95)])
def test_head_sizes_of_65_to_96(size, dtype):
    for layout in ('NTC', 'TNC'):
        d = make(size, dtype, 'cuda:0', layout, seed=11, mask=True,
                 lengths=[size[4], size[4] // 2][:size[0]])
        check(call(d, size, layout, grad=True), oracle(d, size, layout))


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('layout', ['NTC', 'TNC'])
@pytest.mark.parametrize('size', [(2, 2, 1, 0, 5, 8), (2, 2, 1, 3, 0, 8),
                                  (2, 4, 4, 40, 0, 16), (0, 2, 1, 3, 5, 8)])
def test_nothing_to_do_with_values_apart(size, layout, device):
    """An array of no keys has no memory; its attention is zeros."""
    for dtype in TYPES:
        d = make(size, dtype, device, layout, apart=True)
        got = call(d, size, layout, grad=True)
        for g, name in zip(got, ('q', 'q', 'kv', 'values')):
            assert g.shape == d[name].shape and not g.any()


@pytest.mark.gpu
@pytest.mark.parametrize('B', [33, 64, 65, 130])
@pytest.mark.parametrize('heads', [(2, 2), (3, 1), (6, 3)])
@pytest.mark.parametrize('sq', [1, 40])
def test_many_sequences_of_equal_and_unequal_lengths(sq, heads, B):
    """Blocks take the sequences by their lengths, up to 64 of them: each is
    written, once, with ties and empty ones among them."""
    size = (B, *heads, sq, 70, 16)
    g = torch.Generator().manual_seed(B)
    some = torch.randint(0, 75, (B,), generator=g)
    ties = torch.tensor([0, 7, 7, 64, 70])[torch.randint(0, 5, (B,),
                                                         generator=g)]
    for lengths in (some, ties, torch.full((B,), 33), torch.zeros(B),
                    torch.arange(B) % 71, 70 - torch.arange(B) % 71):
        d = make(size, torch.float16, 'cuda:0', seed=12,
                 lengths=lengths.long().tolist())
        check(call(d, size, 'NTC', grad=True), oracle(d, size, 'NTC'))


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('sq,sk', [(1, 70), (40, 70), (3, 3000)])
def test_gradients_that_are_not_finite_beside_no_key(sq, sk, dtype, device):
    """A row without a key is zeros whatever the inputs hold: so is its
    gradient, and other sequences' gradients do not change."""
    size = (3, 4, 2, sq, sk, 32)
    d = make(size, dtype, device, seed=14, lengths=[sk, 0, sk], mask=True)
    d['mask'][2] = False
    want = call(d, size, 'NTC', grad=True)
    for bad in (math.nan, math.inf):
        e = dict(d, dout=d['dout'].clone())
        e['dout'][1:] = bad
        got = call(e, size, 'NTC', grad=True)
        for g, w in zip(got, want):
            assert torch.equal(g[0], w[0])
            assert not g[1:].any() and not w[1:].any()
