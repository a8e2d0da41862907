"""RMSNorm (with the residual's addition, and its int8 output) against the
formula in 64 bits."""
import numpy as np
import pytest
import torch

import mxnet_amd as mx
from mxnet_amd import autograd
from mxnet_amd.gluon import nn

DEVICES = ['cpu', pytest.param('cuda:0', marks=pytest.mark.gpu)]
TYPES = [torch.float16, torch.bfloat16, torch.float32]
U32 = 2.0 ** -24  # half a step of float32


def make(rows, cols, dtype, device, seed=0):
    g = torch.Generator().manual_seed(seed)
    shape = (rows, cols)

    def r(scale=1.0, dt=dtype, sh=shape):
        return (torch.randn(*sh, generator=g) * scale).to(dt).to(device)

    return dict(x=r(), res=r(2.0), gamma=1 + r(0.2, torch.float32, (cols,)),
                dy=r(), dsum=r())


def oracle(x, gamma, res=None, eps=1e-6):
    h = x if res is None else (x.float() + res.float()).to(x.dtype)
    v = h.double()
    r = 1 / torch.sqrt(v.square().mean(-1, keepdim=True) + eps)
    return h, r, v * r * gamma.double()


def half_step(t):
    # relative half step, and the absolute one of the smallest numbers
    f = torch.finfo(t)
    return f.eps / 2, f.smallest_normal * f.eps / 2


def within(got, want, bound):
    bad = (got.double() - want).abs() > bound
    assert not bad.any(), (
        int(bad.sum()), float(((got.double() - want).abs() - bound).max()))


SHAPES = [(1, 1), (1, 8), (3, 7), (5, 64), (32, 1024), (2, 1001), (1, 4099),
          (1500, 768), (1025, 2048), (3, 8192), (2, 20000), (1, 33000),
          (1, 65544)]


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('with_res', [False, True])
@pytest.mark.parametrize('rows,cols', SHAPES)
def test_forward(rows, cols, with_res, dtype, device):
    d = make(rows, cols, dtype, device)
    res = d['res'] if with_res else None
    out = mx.nd.RMSNorm(
        mx.nd.from_torch(d['x']), mx.nd.from_torch(d['gamma']),
        residual=mx.nd.from_torch(res) if with_res else None)
    h, _, want = oracle(d['x'], d['gamma'], res)
    if with_res:
        out, total = out
        assert torch.equal(total.to_torch(), h)
    y = out.to_torch()
    assert y.dtype == dtype and y.shape == d['x'].shape
    # r is rounded once and there are two products: three half steps of
    # float32 (four allow for their own products), then one of the type
    rel, least = half_step(dtype)
    within(y, want, want.abs() * (rel * (1 + 8 * U32) + 4 * U32) + least)


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('with_res', [False, True])
@pytest.mark.parametrize('rows,cols', [(1, 1), (3, 7), (5, 64), (700, 768),
                                       (1030, 1000), (9, 1001), (3, 8192),
                                       (2, 20000), (2, 65544)])
def test_gradient(rows, cols, with_res, dtype, device):
    d = make(rows, cols, dtype, device, seed=1)
    x = mx.nd.from_torch(d['x'].clone().requires_grad_())
    gamma = mx.nd.from_torch(d['gamma'].clone().requires_grad_())
    dy, dsum = d['dy'].double(), d['dsum'].double()
    with autograd.record():
        if with_res:
            res = mx.nd.from_torch(d['res'].clone().requires_grad_())
            y, total = mx.nd.RMSNorm(x, gamma, residual=res)
        else:
            y = mx.nd.RMSNorm(x, gamma)
    if with_res:
        dx, dg, dres = (t.to_torch() for t in autograd.grad(
            [y, total], [x, gamma, res],
            [mx.nd.from_torch(d['dy']), mx.nd.from_torch(d['dsum'])]))
        assert torch.equal(dx, dres)
    else:
        dx, dg = (t.to_torch() for t in autograd.grad(
            [y], [x, gamma], [mx.nd.from_torch(d['dy'])]))
        dsum = torch.zeros_like(dy)
    h, r, _ = oracle(d['x'], d['gamma'], d['res'] if with_res else None)
    g, n = dy * d['gamma'].double(), h.double() * r
    m = (g * n).mean(-1, keepdim=True)
    want = r * (g - n * m) + dsum
    assert dx.dtype == dtype and dg.dtype == torch.float32
    # a thread adds up to 64 products before six to ten levels of a tree; the
    # terms are within that many half steps of float32, each of its own size.
    # On the CPU autograd of the elementary operations rounds dy's path to
    # the type where the norm was, and adds the sum's gradient in the type
    rel, least = half_step(dtype)
    terms = r * g.abs() + r * n.abs() * (
        m.abs() + (g * n).abs().mean(-1, keepdim=True)) + dsum.abs()
    steps = 1 if device != 'cpu' else 4
    within(dx, want, terms * (100 * U32 + (steps - 1) * rel)
           + want.abs() * rel * steps + steps * least)
    # at most ceil(rows / blocks) + 32 + 16 additions in a row
    within(dg, (dy * n).sum(0),
           (dy * n).abs().sum(0) * U32 * (rows + 64) + 1e-30)


def test_gradient_against_differences():
    x = torch.randn(4, 9, dtype=torch.float32)
    res, gamma = torch.randn(4, 9), torch.rand(9) + 0.5
    dy, dsum = torch.randn(4, 9), torch.randn(4, 9)
    xs = mx.nd.from_torch(x.clone().requires_grad_())
    with autograd.record():
        y, h = mx.nd.RMSNorm(xs, mx.nd.from_torch(gamma),
                             residual=mx.nd.from_torch(res))
    dx = autograd.grad([y, h], [xs], [mx.nd.from_torch(dy),
                                      mx.nd.from_torch(dsum)])[0].to_torch()

    def value(v):
        s = v + res.double()
        n = s / torch.sqrt(s.square().mean(-1, keepdim=True) + 1e-6)
        return float((n * gamma.double() * dy).sum() + (s * dsum).sum())

    step = 1e-5
    for at in [(0, 0), (1, 4), (3, 8)]:
        lo, hi = x.double(), x.double()
        lo[at] -= step
        hi[at] += step
        # third derivatives are of the order of 1: the difference is off by
        # about step^2, the gradient by a few half steps of float32
        want = (value(hi) - value(lo)) / (2 * step)
        assert abs(float(dx[at]) - want) < 1e-4


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('with_res', [False, True])
@pytest.mark.parametrize('rows,cols', SHAPES)
def test_int8(rows, cols, with_res, dtype, device):
    d = make(rows, cols, dtype, device, seed=2)
    d['x'][0] *= 30
    res = d['res'] if with_res else None
    out = mx.nd.RMSNorm(
        mx.nd.from_torch(d['x']), mx.nd.from_torch(d['gamma']),
        residual=mx.nd.from_torch(res) if with_res else None,
        out_type='int8')
    h, r, want = oracle(d['x'], d['gamma'], res)
    q, scale = out[0].to_torch(), out[1].to_torch()
    if with_res:
        assert torch.equal(out[2].to_torch(), h)
    assert q.dtype == torch.int8 and scale.shape == (rows, 1)
    # the values, from r rounded to float32 once, are the definition's to the
    # bit: every int8 is the one that the formula gives
    y = h.float() * r.float() * d['gamma']
    top = y.abs().amax(-1, keepdim=True)
    assert torch.equal(scale, top * (1.0 / 127.0))
    inv = torch.reciprocal(top) * 127.0
    assert torch.equal(q, torch.round(y * inv).to(torch.int8))
    # half a step of the scale, and what the factors and products round
    within(q.double() * scale.double(), want,
           scale.double() * (0.5 + 127 * 8 * U32))


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('cols', [64, 1001, 33000])
def test_int8_rows_without_scale(cols, device):
    x = torch.randn(5, cols, device=device)
    x[0] = 0
    x[1, 3] = float('nan')
    x[2, 4] = float('inf')
    x[3, 5] = -float('inf')
    q, scale = mx.nd.RMSNorm(mx.nd.from_torch(x),
                             mx.nd.ones((cols,), ctx=mx.gpu(0) if device
                                        != 'cpu' else mx.cpu()),
                             out_type='int8')
    q, scale = q.to_torch().cpu(), scale.to_torch().cpu()
    assert not q[:4].any() and float(scale[0]) == 1.0
    assert torch.isnan(scale[1:4]).all()
    assert int(q[4].abs().max()) == 127 and float(scale[4]) > 0


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', TYPES)
def test_views_on_the_gpu(dtype):
    """Strided and misaligned inputs give what their copies give."""
    big = torch.randn(40, 1030, device='cuda:0').to(dtype)
    gamma = torch.rand(1024, device='cuda:0')
    x, res = big[::2, 3:1027], big[1::2, 1:1025]
    a = mx.nd.RMSNorm(mx.nd.from_torch(x), mx.nd.from_torch(gamma),
                      residual=mx.nd.from_torch(res))
    flat = torch.empty(20 * 1024 + 1, device='cuda:0', dtype=dtype)
    odd = flat[1:].view(20, 1024)
    odd.copy_(x)
    b = mx.nd.RMSNorm(mx.nd.from_torch(odd), mx.nd.from_torch(gamma),
                      residual=mx.nd.from_torch(res.contiguous()))
    h, _, want = oracle(x, gamma, res)
    rel, least = half_step(dtype)
    for y, total in (a, b):
        assert torch.equal(total.to_torch(), h)
        within(y.to_torch(), want,
               want.abs() * (rel * (1 + 8 * U32) + 4 * U32) + least)


@pytest.mark.gpu
def test_other_stream_and_graph():
    d = make(64, 768, torch.float16, 'cuda:0', seed=3)
    nd = mx.nd.from_torch
    want = mx.nd.RMSNorm(nd(d['x']), nd(d['gamma']), residual=nd(d['res']))
    want = [t.to_torch().clone() for t in want]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = mx.nd.RMSNorm(nd(d['x']), nd(d['gamma']), residual=nd(d['res']))
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(got, want):
        assert torch.equal(a.to_torch(), b)
    graph = torch.cuda.CUDAGraph()
    with torch.no_grad(), torch.cuda.graph(graph):
        y, h = mx.nd.RMSNorm(nd(d['x']), nd(d['gamma']),
                             residual=nd(d['res']))
    for k in range(3):
        d['x'].copy_(make(64, 768, torch.float16, 'cuda:0', seed=10 + k)['x'])
        graph.replay()
        torch.cuda.synchronize()
        e = mx.nd.RMSNorm(nd(d['x']), nd(d['gamma']), residual=nd(d['res']))
        assert torch.equal(y.to_torch(), e[0].to_torch())
        assert torch.equal(h.to_torch(), e[1].to_torch())


@pytest.mark.parametrize('device', DEVICES)
def test_empty_and_unused(device):
    x = torch.empty(0, 16, device=device, requires_grad=True)
    gamma = torch.ones(16, device=device, requires_grad=True)
    with autograd.record():
        y = mx.nd.RMSNorm(mx.nd.from_torch(x), mx.nd.from_torch(gamma))
    assert y.shape == (0, 16)
    q, scale = mx.nd.RMSNorm(mx.nd.from_torch(x.detach()),
                             mx.nd.from_torch(gamma.detach()),
                             out_type='int8')
    assert q.shape == (0, 16) and scale.shape == (0, 1)
    # a loss of the sum alone
    x = torch.randn(3, 16, device=device, requires_grad=True)
    res = torch.randn(3, 16, device=device, requires_grad=True)
    with autograd.record():
        _, h = mx.nd.RMSNorm(mx.nd.from_torch(x), mx.nd.from_torch(gamma),
                             residual=mx.nd.from_torch(res))
        h.backward()
    assert torch.equal(x.grad, torch.ones_like(x))
    assert torch.equal(res.grad, torch.ones_like(x))


def test_refusals():
    nd = mx.nd.from_torch
    x, gamma = torch.randn(2, 8), torch.ones(8)
    with pytest.raises(TypeError):
        mx.nd.RMSNorm(nd(x.double()), nd(gamma))
    with pytest.raises(ValueError):
        mx.nd.RMSNorm(nd(x), nd(torch.ones(7)))
    with pytest.raises(ValueError):
        mx.nd.RMSNorm(nd(x), nd(gamma), residual=nd(x[:1]))
    with pytest.raises(ValueError):
        mx.nd.RMSNorm(nd(x), nd(gamma), residual=nd(x.half()))
    with pytest.raises(ValueError):
        mx.nd.RMSNorm(nd(x), nd(gamma), out_type='uint8')
    with pytest.raises(NotImplementedError):
        mx.nd.RMSNorm(nd(x), nd(gamma), axis=0)
    with pytest.raises(ValueError):
        with autograd.record():
            mx.nd.RMSNorm(nd(x.clone().requires_grad_()), nd(gamma),
                          out_type='int8')


def test_gluon_layer_and_symbol(tmp_path):
    layer = nn.RMSNorm(epsilon=1e-5)
    layer.initialize()
    x, res = mx.nd.array(np.random.randn(3, 12)), \
        mx.nd.array(np.random.randn(3, 12))
    y = layer(x)
    _, _, want = oracle(x.to_torch(), torch.ones(12), eps=1e-5)
    within(y.to_torch(), want, want.abs() * 16 * U32)
    y2, h = layer(x, res)
    assert torch.equal(h.to_torch(), x.to_torch() + res.to_torch())
    layer.cast('float16')
    assert layer.gamma.data().dtype == np.float32
    a, b, g = (mx.sym.var(n) for n in 'abg')
    feed = {'a': x, 'b': res, 'g': mx.nd.ones((12,))}
    ys, hs = mx.sym.RMSNorm(a, g, residual=b, eps=1e-5)
    net = mx.sym.Group([ys, hs])
    got = net.eval_dict(feed)
    assert torch.equal(got[0].to_torch(), y2.to_torch())
    assert torch.equal(got[1].to_torch(), h.to_torch())
    net.save(str(tmp_path / 'n.json'))
    got = mx.sym.load(str(tmp_path / 'n.json')).eval_dict(feed)
    assert torch.equal(got[0].to_torch(), y2.to_torch())
    assert torch.equal(mx.sym.RMSNorm(a, g, eps=1e-5).eval_dict(feed)[0]
                       .to_torch(), y.to_torch())


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('cols', [64, 1001, 33000])
@pytest.mark.parametrize('value', [float('nan'), float('inf')])
def test_int8_of_a_gamma_that_is_not_finite(value, cols, device):
    """No row can be scaled then: a finite scale would hide the value."""
    x = torch.randn(3, cols, device=device)
    gamma = torch.ones(cols, device=device)
    gamma[cols // 2] = value
    q, scale = mx.nd.RMSNorm(mx.nd.from_torch(x), mx.nd.from_torch(gamma),
                             out_type='int8')
    assert torch.isnan(scale.to_torch()).all() and not q.to_torch().any()


@pytest.mark.gpu
@pytest.mark.parametrize('out_type', [None, 'int8'])
def test_more_rows_than_one_launch_takes(out_type):
    """2^32 threads or more are not one launch: 2^23 rows of a wave each."""
    x = torch.randn((1 << 23) + 5, 1, device='cuda:0').half()
    res = torch.randn((1 << 23) + 5, 1, device='cuda:0').half()
    gamma = torch.full((1,), 0.75, device='cuda:0')
    out = mx.nd.RMSNorm(mx.nd.from_torch(x), mx.nd.from_torch(gamma),
                        residual=mx.nd.from_torch(res), out_type=out_type)
    h, r, want = oracle(x, gamma, res)
    assert torch.equal(out[-1].to_torch(), h)
    if out_type is None:
        rel, least = half_step(torch.float16)
        within(out[0].to_torch(), want,
               want.abs() * (rel * (1 + 8 * U32) + 4 * U32) + least)
    else:
        y = h.float() * r.float() * gamma
        q, scale = out[0].to_torch(), out[1].to_torch()
        assert torch.equal(q, 127 * torch.sign(y).to(torch.int8))
        some = torch.where(y == 0, 1.0, y.abs() * (1.0 / 127.0))
        assert torch.equal(scale, some)


@pytest.mark.gpu
def test_past_2_31_elements():
    """The last rows of 4 GB give what they give alone, forward and back."""
    rows, cols = (1 << 19) + 6, 4096
    d = make(6, cols, torch.bfloat16, 'cuda:0', seed=5)
    big = torch.zeros(rows, cols, dtype=torch.bfloat16, device='cuda:0')
    dy = torch.zeros_like(big)
    big[-6:], dy[-6:] = d['x'], d['dy']
    both = []
    for x, g in ((d['x'], d['dy']), (big, dy)):
        x, gamma = (mx.nd.from_torch(t.detach().requires_grad_())
                    for t in (x, d['gamma']))
        with autograd.record():
            y = mx.nd.RMSNorm(x, gamma)
        dx, dg = autograd.grad([y], [x, gamma], [mx.nd.from_torch(g)])
        both.append((y.to_torch()[-6:].detach().clone(),
                     dx.to_torch()[-6:].clone(), dg.to_torch()))
    (y0, dx0, dg0), (y1, dx1, dg1) = both
    # (few rows take a block each, many a wave: other orders of 32-bit sums)
    rel, least = half_step(torch.bfloat16)
    assert torch.equal(y0, y1)
    for a, b, scale in ((dx0, dx1, 1.0), (dg0, dg1, 0.0)):
        a, b = a.double(), b.double()
        size = a.abs().amax()
        within(a, b, a.abs() * 2 * rel * scale + size * cols * 4 * U32 + least)


@pytest.mark.gpu
def test_second_derivatives_are_refused():
    d = make(4, 64, torch.float32, 'cuda:0', seed=6)
    x = d['x'].requires_grad_()
    with autograd.record():
        y = mx.nd.RMSNorm(mx.nd.from_torch(x), mx.nd.from_torch(d['gamma']))
    dx, = autograd.grad([y], [mx.nd.from_torch(x)], create_graph=True,
                        retain_graph=True)
    with pytest.raises(RuntimeError):
        dx.to_torch().square().sum().backward()


@pytest.mark.gpu
def test_gradient_of_many_rows():
    """dgamma's partials of twice as many blocks; sums of 16400 products of
    values of order one in 32 bits, in an order of the kernel's own."""
    rows, cols = 16400, 64
    d = make(rows, cols, torch.float32, 'cuda:0', seed=14)
    x, gamma = (mx.nd.from_torch(d[k].requires_grad_()) for k in ('x', 'gamma'))
    with autograd.record():
        y = mx.nd.RMSNorm(x, gamma)
    dx, dg = autograd.grad([y], [x, gamma], [mx.nd.from_torch(d['dy'])])
    h, g, dy = (d[k].detach().double() for k in ('x', 'gamma', 'dy'))
    r = 1 / torch.sqrt(h.square().mean(-1, keepdim=True) + 1e-6)
    n, t = h * r, dy * g
    want = r * (t - n * (t * n).mean(-1, keepdim=True))
    within(dx.to_torch(), want, r * (t.abs() + n.abs() * (
        t * n).abs().mean(-1, keepdim=True)) * (cols + 8) * U32)
    within(dg.to_torch(), (dy * n).sum(0), (dy * n).abs().sum(0)
           * (rows + 8) * U32)


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('with_res', [False, True])
@pytest.mark.parametrize('rows,cols', [(3, 12288), (600, 9000), (2, 20000),
                                       (5, 32768), (3, 9001)])
def test_wide_rows(rows, cols, with_res, dtype):
    """A block of 1024 threads a row, with one row ahead or without."""
    test_forward(rows, cols, with_res, dtype, 'cuda:0')
    test_gradient(rows, cols, with_res, dtype, 'cuda:0')


@pytest.mark.gpu
def test_captured_backward():
    d = make(64, 768, torch.float16, 'cuda:0', seed=15)

    def call():
        x, res, gamma = (mx.nd.from_torch(d[k].detach().requires_grad_())
                         for k in ('x', 'res', 'gamma'))
        with autograd.record():
            y, h = mx.nd.RMSNorm(x, gamma, residual=res)
        grads = autograd.grad([y, h], [x, res, gamma],
                              [mx.nd.from_torch(d[k]) for k in ('dy', 'dsum')])
        return [t.to_torch().detach() for t in [y, h] + grads]

    call()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        caught = call()
    for k in range(3):
        e = make(64, 768, torch.float16, 'cuda:0', seed=30 + k)
        for name in ('x', 'res', 'dy', 'dsum'):
            d[name].copy_(e[name])
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(caught, call()):
            assert torch.equal(a, b)


def test_a_tangent_is_seen():
    from mxnet_amd.ops.nn import needs_grad
    x = torch.randn(3, 8)
    assert not needs_grad(x, None)
    with torch.autograd.forward_ad.dual_level():
        assert not needs_grad(x, None)
        dual = torch.autograd.forward_ad.make_dual(x, torch.ones_like(x))
        assert needs_grad(None, dual)
        with torch.no_grad():  # which leaves forward mode on
            assert needs_grad(dual)


@pytest.mark.gpu
def test_forward_mode_is_refused_on_the_gpu():
    """There is no kernel for tangents: refused, not dropped."""
    x = torch.randn(3, 8, device='cuda:0')
    one = torch.ones(8, device='cuda:0')
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(x, torch.ones_like(x))
        for data, gamma, res in ((dual, one, None), (x, one, dual),
                                 (x, torch.autograd.forward_ad.make_dual(
                                     one, one), None)):
            with pytest.raises(RuntimeError):
                mx.nd.RMSNorm(*(mx.nd.from_torch(t) for t in (data, gamma)),
                              residual=None if res is None
                              else mx.nd.from_torch(res))
        with pytest.raises(ValueError):
            mx.nd.RMSNorm(mx.nd.from_torch(dual), mx.nd.from_torch(one),
                          out_type='int8')
        kv = mx.nd.from_torch(torch.randn(1, 4, 16, device='cuda:0'))
        with pytest.raises(RuntimeError):
            mx.nd.contrib.encdec_attention(mx.nd.from_torch(dual[None]), kv)


@pytest.mark.gpu
def test_gradients_of_rows_past_2_27_columns():
    """More columns than one launch of dgamma's last sum has threads for."""
    rows, cols = 2, (1 << 27) + 3
    g = torch.Generator(device='cuda:0').manual_seed(41)
    x, dy = (torch.randn(rows, cols, device='cuda:0', generator=g).bfloat16()
             for _ in range(2))
    gamma = torch.rand(cols, device='cuda:0', generator=g) + 0.5
    xs, gs = (mx.nd.from_torch(t.requires_grad_()) for t in (x, gamma))
    with autograd.record():
        y = mx.nd.RMSNorm(xs, gs)
    dx, dg = (t.to_torch() for t in autograd.grad(
        [y], [xs, gs], [mx.nd.from_torch(dy)]))
    r = torch.rsqrt(torch.stack([t.double().square().mean() for t in x.detach()])
                    + 1e-6)[:, None]
    m = torch.stack([(a.double() * gamma.detach() * b).sum()
                     for a, b in zip(dy, x.detach())])[:, None] * r / cols
    for at in (slice(0, 1000), slice((1 << 26) - 500, (1 << 26) + 500),
               slice(cols - 1000, cols)):
        n = x.detach()[:, at].double() * r
        a = dy[:, at].double()
        # two products, each of two rounded factors, and their sum
        within(dg[at], (a * n).sum(0), (a * n).abs().sum(0) * U32 * 6 + 1e-30)
        t = a * gamma.detach()[at].double()
        want = r * (t - n * m)
        # (m is the mean of 2^27 terms: off by 2^-7 of their size at most, of
        # which the row's sum of 2^17 in a thread has half a step each)
        off = r * (t.abs() * 4 * U32 + n.abs() * (m.abs() * 8 * U32
                                                  + 2.0 ** 17 * U32))
        within(dx[:, at], want, off + want.abs() * 2.0 ** -8 + 1e-30)
