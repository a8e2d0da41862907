"""RMSNorm, encdec_attention and sample_tokens on the native runtime, and a
run of the three together on both."""
import numpy as np
import pytest
import torch

import mxnet_amd as mx
from mxnet_amd import autograd
from mxnet_amd.base import set_native
from mxnet_amd.gluon import nn

DEVICES = ['cpu', pytest.param('gpu', marks=pytest.mark.gpu)]


@pytest.fixture
def native():
    prev = set_native(True)
    yield
    set_native(prev)


def ctx(device):
    return mx.cpu() if device == 'cpu' else mx.gpu(0)


def arr(a, device, dtype=None):
    x = mx.nd.array(a, ctx=ctx(device), dtype=str(a.dtype))
    assert x.is_native
    return x if dtype is None else x.astype(dtype)


def near(got, want, dtype='float32'):
    # float32: sums of some hundred products, of values of order one; half
    # types: three roundings on the way, of terms a few times the result
    tol = {'float32': 1e-5, 'float16': 4 * 2.0 ** -11}[dtype]
    got, want = got.asnumpy().astype('float64'), want.astype('float64')
    assert got.shape == want.shape
    assert np.abs(got - want).max(initial=0) <= tol * (
        1 + np.abs(want).max(initial=0))


def torch_rms(x, g, res, dy, dsum):
    x, g = (torch.tensor(t, dtype=torch.float64, requires_grad=True)
            for t in (x, g))
    h = x if res is None else x + torch.tensor(res, dtype=torch.float64)
    y = h / torch.sqrt(h.square().mean(-1, keepdim=True) + 1e-6) * g
    loss = (y * torch.tensor(dy)).sum()
    if res is not None:
        loss = loss + (h * torch.tensor(dsum)).sum()
    loss.backward()
    return [t.detach().numpy() for t in (y, h, x.grad, g.grad)]


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('with_res', [False, True])
@pytest.mark.parametrize('shape', [(3, 7), (2, 5, 64), (600, 256)])
def test_rms_norm(native, shape, with_res, device):
    rs = np.random.RandomState(0)
    x, res, dy, dsum = (rs.randn(*shape).astype('float32') for _ in range(4))
    g = (1 + 0.2 * rs.randn(shape[-1])).astype('float32')
    xs, gs, rr = arr(x, device), arr(g, device), arr(res, device)
    for v in (xs, gs, rr):
        v.attach_grad()
    with autograd.record():
        if with_res:
            y, h = mx.nd.RMSNorm(xs, gs, residual=rr)
            loss = (y * arr(dy, device)).sum() + (h * arr(dsum, device)).sum()
        else:
            y = mx.nd.RMSNorm(xs, gs)
            loss = (y * arr(dy, device)).sum()
    loss.backward()
    want = torch_rms(x, g, res if with_res else None, dy, dsum)
    near(y, want[0])
    near(xs.grad, want[2])
    near(gs.grad, want[3])
    if with_res:
        near(h, want[1])
        near(rr.grad, want[2])


@pytest.mark.parametrize('device', DEVICES)
def test_rms_norm_of_the_sum_alone(native, device):
    x = np.random.RandomState(1).randn(3, 16).astype('float32')
    xs, rr, g = arr(x, device), arr(x, device), arr(np.ones(16, 'float32'),
                                                    device)
    xs.attach_grad()
    rr.attach_grad()
    with autograd.record():
        _, h = mx.nd.RMSNorm(xs, g, residual=rr)
        loss = h.sum()
    loss.backward()
    assert np.array_equal(xs.grad.asnumpy(), np.ones_like(x))
    assert np.array_equal(rr.grad.asnumpy(), np.ones_like(x))


@pytest.mark.parametrize('device', DEVICES)
def test_rms_norm_int8(native, device):
    rs = np.random.RandomState(2)
    x, res = (rs.randn(9, 100).astype('float32') for _ in range(2))
    x[1], res[1] = 0, 0
    x[2, 3] = np.nan
    g = (1 + 0.2 * rs.randn(100)).astype('float32')
    q, s, h = mx.nd.RMSNorm(arr(x, device), arr(g, device),
                            residual=arr(res, device), out_type='int8')
    set_native(False)
    want = mx.nd.RMSNorm(*(mx.nd.from_torch(torch.tensor(t)) for t in (x, g)),
                         residual=mx.nd.from_torch(torch.tensor(res)),
                         out_type='int8')
    set_native(True)
    assert np.array_equal(q.asnumpy(), want[0].asnumpy())
    assert np.array_equal(s.asnumpy(), want[1].asnumpy(), equal_nan=True)
    assert np.array_equal(h.asnumpy(), want[2].asnumpy(), equal_nan=True)


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('apart', [False, True])
@pytest.mark.parametrize('layout', ['NTC', 'TNC'])
@pytest.mark.parametrize('sq', [1, 70])
def test_attention(native, sq, layout, apart, device):
    """Against the torch frontend's CPU path, gradients among it."""
    rs = np.random.RandomState(3)
    B, H, Hk, sk, D = 3, 4, 2, 90, 16

    def r(s, w):
        return rs.randn(*((B, s, w) if layout == 'NTC' else (s, B, w))) \
            .astype('float32')

    q, dout = r(sq, H * D), r(sq, H * D)
    kvs = [r(sk, Hk * D), r(sk, Hk * D)] if apart else [r(sk, 2 * Hk * D)]
    length = np.array([40, 0, 90], 'int64')
    mask = (rs.rand(B, sk) < 0.7).astype('uint8')
    kw = dict(heads=H, kv_heads=Hk, layout=layout)
    ins = [arr(v, device) for v in [q] + kvs]
    for v in ins:
        v.attach_grad()
    with autograd.record():
        out = mx.nd.contrib.encdec_attention(
            *ins, valid_length=arr(length, device), mask=arr(mask, device),
            **kw)
        loss = (out * arr(dout, device)).sum()
    loss.backward()
    set_native(False)
    ts = [mx.nd.from_torch(torch.tensor(v, requires_grad=True))
          for v in [q] + kvs]
    with autograd.record():
        want = mx.nd.contrib.encdec_attention(
            *ts, valid_length=mx.nd.from_torch(torch.tensor(length)),
            mask=mx.nd.from_torch(torch.tensor(mask)), **kw)
    grads = autograd.grad([want], ts, [mx.nd.from_torch(torch.tensor(dout))])
    set_native(True)
    near(out, want.to_torch().detach().numpy())
    for v, g in zip(ins, grads):
        near(v.grad, g.asnumpy())


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('v', [50, 20000])
def test_sample(native, v, device):
    rs = np.random.RandomState(4)
    x = (2.5 * rs.randn(5, v)).astype('float32')
    x[3] = -np.inf
    u = rs.rand(5).astype('float32')
    rows = dict(temperature=np.array([0.5, 1, 0, 2, 1], 'float32'),
                top_k=np.array([0, 5, 3, 1, 40], 'int32'),
                top_p=np.array([0.9, 1, 1, 1, 0.5], 'float32'),
                min_p=np.array([0, 0.1, 0, 0, 0.01], 'float32'))
    for kw in (dict(temperature=0.7, top_k=40, top_p=0.9), dict(min_p=0.1),
               rows):
        def both(make):
            return mx.nd.contrib.sample_tokens(
                make(x), make(u), get_prob=True,
                **{k: make(p) if isinstance(p, np.ndarray) else p
                   for k, p in kw.items()})
        t, lp = both(lambda a: arr(a, device))
        set_native(False)
        wt, wlp = both(lambda a: mx.nd.from_torch(torch.tensor(a)))
        set_native(True)
        assert np.array_equal(t.asnumpy(), wt.asnumpy())
        assert np.allclose(lp.asnumpy(), wlp.asnumpy(), rtol=2.0 ** -22,
                           atol=1e-9, equal_nan=True)


def test_refusals(native):
    def a(*shape):
        return arr(np.zeros(shape, 'float32'), 'cpu')

    with pytest.raises(RuntimeError):
        mx.nd.RMSNorm(a(2, 8), a(7))
    with pytest.raises(RuntimeError):
        mx.nd.RMSNorm(a(2, 8), a(8), residual=a(1, 8))
    with pytest.raises(ValueError):
        mx.nd.RMSNorm(a(2, 8), a(8), out_type='uint8')
    with pytest.raises(NotImplementedError):
        mx.nd.RMSNorm(a(2, 8), a(8), axis=0)
    f = mx.nd.contrib.encdec_attention
    with pytest.raises(RuntimeError):
        f(a(1, 2, 8), a(1, 3, 8), heads=2)
    with pytest.raises(RuntimeError):
        f(a(1, 2, 8), a(1, 3, 16), heads=3)
    with pytest.raises(RuntimeError):
        f(a(1, 2, 8), a(1, 3, 16), heads=2, valid_length=a(1))
    with pytest.raises(RuntimeError):
        f(a(1, 2, 8), a(1, 3, 16), heads=2, mask=a(1, 3))
    with pytest.raises(ValueError):
        f(a(1, 2, 8), a(1, 3, 16), heads=2, layout='CTN')
    g = mx.nd.contrib.sample_tokens
    with pytest.raises(RuntimeError):
        g(a(2, 8), a(3))
    with pytest.raises(RuntimeError):
        g(a(2, 8), a(2), top_p=a(3))
    with pytest.raises(ValueError):
        g(a(2, 8), a(2), top_p=1.5)


# -- the three together -------------------------------------------------------

class Layer(nn.HybridBlock):
    """What a decoder layer does with an encoder's states: norm, attention
    over them, residual and norm again."""

    def __init__(self, units, heads, **kw):
        super().__init__(**kw)
        self.heads = heads
        self.norm1, self.norm2 = nn.RMSNorm(), nn.RMSNorm()
        self.query = nn.Dense(units, flatten=False, in_units=units)
        self.key_value = nn.Dense(2 * units, flatten=False, in_units=units)
        self.proj = nn.Dense(units, flatten=False, in_units=units)

    def forward(self, x, states, valid_length):
        a = mx.nd.contrib.encdec_attention(
            self.query(self.norm1(x)), self.key_value(states),
            heads=self.heads, valid_length=valid_length)
        return self.norm2(self.proj(a), x)


def step(device, weights, data, train, dtype='float32'):
    net = Layer(64, 4)
    net.initialize(ctx=ctx(device))
    net.cast(dtype)
    x, states, length, head, u = data
    xs = arr2(x, device, dtype)
    net(xs, arr2(states, device, dtype), arr2(length, device))
    for (_, p), w in zip(sorted(net.collect_params().items()), weights):
        p.set_data(arr2(w, device, str(p.data().dtype)))
    with autograd.record():
        y, h = net(xs, arr2(states, device, dtype), arr2(length, device))
        loss = (y * h).sum()
    if train:
        loss.backward()
        return [y, h] + [p.grad() for _, p in
                         sorted(net.collect_params().items())]
    logits = mx.nd.FullyConnected(y[:, -1], arr2(head, device, dtype),
                                  no_bias=True, num_hidden=head.shape[0])
    return [mx.nd.contrib.sample_tokens(logits, arr2(u, device), top_k=20,
                                        top_p=0.9)]


def arr2(a, device, dtype=None):
    x = mx.nd.array(a, ctx=ctx(device), dtype=str(a.dtype))
    return x if dtype in (None, str(a.dtype)) else x.astype(dtype)


def inputs(sq):
    rs = np.random.RandomState(5)
    data = [rs.randn(3, sq, 64).astype('float32'),
            rs.randn(3, 50, 64).astype('float32'),
            np.array([50, 17, 0], 'int32'),
            rs.randn(300, 64).astype('float32'),
            rs.rand(3).astype('float32')]
    net = Layer(64, 4)
    net.initialize()
    shapes = []
    with autograd.pause():
        net(arr2(data[0], 'cpu'), arr2(data[1], 'cpu'), arr2(data[2], 'cpu'))
    for _, p in sorted(net.collect_params().items()):
        shapes.append(tuple(p.shape))
    return data, [(0.1 * rs.randn(*s) + (len(s) == 1)).astype('float32')
                  for s in shapes]


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('on_native', [False, True])
def test_training_and_drawing_together(on_native, device):
    """Gradients of the layer, and the tokens drawn behind it, are the CPU
    path's on either runtime and device."""
    prev = set_native(False)
    try:
        data, weights = inputs(5)
        want = [t.asnumpy() for t in step('cpu', weights, data, True)]
        tokens = step('cpu', weights, data, False)[0].asnumpy()
        set_native(on_native)
        got = step(device, weights, data, True)
        for g, w in zip(got, want):
            g, w = g.asnumpy().astype('float64'), w.astype('float64')
            # sums of up to 960 products in float32 behind two others
            assert np.abs(g - w).max() <= 2e-4 * (1 + np.abs(w).max())
        assert np.array_equal(
            step(device, weights, data, False)[0].asnumpy(), tokens)
    finally:
        set_native(prev)


@pytest.mark.gpu
def test_int8_product_behind_the_norm():
    """The int8 output feeds the int8 product: one scale a row on one side,
    one for the weight on the other."""
    from mxnet_amd.ops import hipshim as ext
    g = torch.Generator(device='cuda:0').manual_seed(0)
    x, res = (torch.randn(70, 256, device='cuda:0', generator=g).half()
              for _ in range(2))
    gamma = torch.rand(256, device='cuda:0', generator=g) + 0.5
    w = torch.randint(-127, 128, (128, 256), device='cuda:0',
                      generator=g).to(torch.int8)
    nd = mx.nd.from_torch
    q, s, h = mx.nd.RMSNorm(nd(x), nd(gamma), residual=nd(res),
                            out_type='int8')
    out = ext.gemm_nt_i8(q.to_torch(), w, 0.01, torch.float32) * s.to_torch()
    v = h.to_torch().double()
    y = v / torch.sqrt(v.square().mean(-1, keepdim=True) + 1e-6) * gamma
    # each of 256 values is off by half a step of its row's scale at most
    wd = w.double() * 0.01
    off = 0.5 * s.to_torch().double() * wd.abs().sum(1)[None]
    assert ((out.double() - y @ wd.T).abs() <= off * 1.01).all()


@pytest.mark.parametrize('device', DEVICES)
def test_int8_of_a_gamma_that_is_not_finite(native, device):
    x = np.random.RandomState(11).randn(3, 40).astype('float32')
    for value in (np.nan, np.inf):
        g = np.ones(40, 'float32')
        g[7] = value
        q, scale = mx.nd.RMSNorm(arr(x, device), arr(g, device),
                                 out_type='int8')
        assert np.isnan(scale.asnumpy()).all() and not q.asnumpy().any()


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', ['float16', 'bfloat16', 'float32'])
def test_both_frontends_run_one_kernel(native, dtype):
    """The native runtime gives the torch frontend's results to the bit, with
    workspaces (split keys, rows in parts) among them."""
    rs = np.random.RandomState(12)
    tt = getattr(torch, dtype)

    def pair(*shape, grad=False):
        a = rs.randn(*shape).astype('float32')
        n = mx.nd.array(a, ctx=mx.gpu(0), dtype='float32').astype(dtype)
        t = torch.tensor(a, device='cuda:0').to(tt).requires_grad_(grad)
        return n, mx.nd.from_torch(t)

    def same(n, t):
        n = n.astype('float32').asnumpy()
        assert np.array_equal(n, t.to_torch().detach().float().cpu().numpy())

    # (dout: what the loss passes down, the same in both)
    q, k, dout = pair(2, 3, 256, grad=True), pair(2, 5000, 256, grad=True), \
        pair(2, 3, 256)
    x, res = pair(70, 256, grad=True), pair(70, 256, grad=True)
    gamma = rs.rand(256).astype('float32')
    gn = mx.nd.array(gamma, ctx=mx.gpu(0), dtype='float32')
    gt = mx.nd.from_torch(torch.tensor(gamma, device='cuda:0',
                                       requires_grad=True))
    z, u = pair(3, 60000), rs.rand(3).astype('float32')
    kw = dict(heads=8, kv_heads=4)
    for v in (q[0], k[0], x[0], res[0], gn):
        v.attach_grad()
    with autograd.record():
        on = mx.nd.contrib.encdec_attention(q[0], k[0], **kw)
        yn, hn = mx.nd.RMSNorm(x[0], gn, residual=res[0])
    autograd.backward([on, yn, hn], [dout[0], x[0], res[0]])
    tn = mx.nd.contrib.sample_tokens(z[0], mx.nd.array(u, ctx=mx.gpu(0)),
                                     top_p=0.8)
    set_native(False)
    with autograd.record():
        ot = mx.nd.contrib.encdec_attention(q[1], k[1], **kw)
        yt, ht = mx.nd.RMSNorm(x[1], gt, residual=res[1])
    gq, gk = autograd.grad([ot], [q[1], k[1]], [dout[1]])
    gx, gg = autograd.grad([yt, ht], [x[1], gt],
                           [mx.nd.from_torch(v.to_torch().detach())
                            for v in (x[1], res[1])])
    t = mx.nd.contrib.sample_tokens(
        z[1], mx.nd.from_torch(torch.tensor(u, device='cuda:0')), top_p=0.8)
    same(on, ot)
    same(yn, yt)
    same(hn, ht)
    same(q[0].grad, gq)
    same(k[0].grad, gk)
    same(x[0].grad, gx)
    same(res[0].grad, gx)
    same(gn.grad, gg)
    same(tn, t)
    set_native(True)


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('sq', [1, 40])
def test_lengths_that_int32_does_not_hold(native, sq, device):
    """int64 lengths mean what the same lengths within the keys mean, also
    where neither int32 nor float32 holds them."""
    rs = np.random.RandomState(13)
    far = [(1 << 40), (1 << 63) - 1, -(1 << 40), (1 << 32) + 2, 1 << 31,
           -(1 << 63), 4]
    near_by = [9, 9, 0, 9, 9, 0, 4]
    q, dout = (rs.randn(7, sq, 16).astype('float32') for _ in range(2))
    kv = rs.randn(7, 9, 16).astype('float32')
    got = []
    for length, dtype in ((far, 'int64'), (near_by, 'int64'),
                          (near_by, 'int32')):
        ins = [arr(q, device), arr(kv, device)]
        for v in ins:
            v.attach_grad()
        with autograd.record():
            out = mx.nd.contrib.encdec_attention(
                *ins, heads=2, kv_heads=1,
                valid_length=arr(np.array(length, dtype), device))
        autograd.backward([out], [arr(dout, device)])
        got.append([t.asnumpy() for t in [out] + [v.grad for v in ins]])
    for a, b, c in zip(*got):
        assert np.array_equal(a, c) and np.array_equal(b, c)
    assert np.abs(got[0][0]).max((1, 2))[[0, 1, 3, 4, 6]].all()


@pytest.mark.parametrize('device', DEVICES)
def test_types_of_sampling_parameters(native, device):
    """The torch frontend's rules: parameters of the wrong kind are refused,
    the others' values count, whatever their size."""
    rs = np.random.RandomState(14)
    x, u = arr(rs.randn(6, 30).astype('float32'), device), \
        arr(rs.rand(6).astype('float32'), device)
    f = mx.nd.contrib.sample_tokens
    with pytest.raises(TypeError):
        f(x, u, top_k=arr(np.full(6, 1.9, 'float32'), device))
    for name in ('temperature', 'top_p', 'min_p'):
        with pytest.raises(TypeError):
            f(x, u, **{name: arr(np.ones(6, 'int32'), device)})
    want = f(x, u, top_k=arr(np.array([0, 1, 5, 0, 30, 0], 'int32'), device))
    # (of no limit, 1, 5, no limit, as many as there are and less than none)
    far = np.array([1 << 32, 1, 5, (1 << 63) - 1, 30, -(1 << 40)], 'int64')
    assert np.array_equal(f(x, u, top_k=arr(far, device)).asnumpy(),
                          want.asnumpy())
    for kind in ('int8', 'uint8', 'int64'):
        got = f(x, u, top_k=arr(np.array([0, 1, 5, 0, 30, 0], kind), device))
        assert np.array_equal(got.asnumpy(), want.asnumpy())
    t = np.array([0.5, 1, 0, 2, 1, 0.25])
    want = f(x, u, temperature=arr(t.astype('float32'), device))
    for kind in ('float16', 'float64'):
        got = f(x, u, temperature=arr(t.astype(kind), device))
        assert np.array_equal(got.asnumpy(), want.asnumpy())


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('apart', [False, True])
def test_attention_over_no_keys(native, apart, device):
    q = np.ones((2, 3, 16), 'float32')
    ins = [arr(q, device)] + [
        mx.nd.zeros((2, 0, 8 if apart else 16), ctx=ctx(device))
        for _ in range(2 if apart else 1)]
    for v in ins:
        v.attach_grad()
    with autograd.record():
        out = mx.nd.contrib.encdec_attention(*ins, heads=4, kv_heads=2)
    autograd.backward([out], [arr(q, device)])
    assert out.shape == q.shape and not out.asnumpy().any()
    for v in ins:
        assert v.grad.shape == v.shape and not v.grad.asnumpy().any()


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('on_native', [False, True])
def test_int8_output_where_a_gradient_would_follow(on_native, device):
    """Refused at the call on both runtimes, for marked arrays and for what
    was computed of them; other calls within record() pass."""
    prev = set_native(on_native)
    try:
        x, g = (mx.nd.array(np.ones(s, 'float32'), ctx=ctx(device))
                for s in ((2, 16), (16,)))
        assert x.is_native == on_native
        free = mx.nd.array(np.ones((2, 16), 'float32'), ctx=ctx(device))
        x.attach_grad()
        with autograd.record():
            for args in ((x, g, None), (x * 2, g, None), (free, g, x),
                         (free, g, free + x)):
                with pytest.raises(ValueError):
                    mx.nd.RMSNorm(args[0], args[1], residual=args[2],
                                  out_type='int8')
            q = mx.nd.RMSNorm(free, g, residual=free * 2, out_type='int8')[0]
        assert (q.asnumpy() == 127).all()
    finally:
        set_native(prev)


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('on_native', [False, True])
def test_int8_output_of_a_trained_layer(on_native, device):
    """Outside record() a layer's gamma and marked arrays give int8, as no
    gradient follows."""
    prev = set_native(on_native)
    try:
        layer = nn.RMSNorm()
        layer.initialize(ctx=ctx(device))
        x = mx.nd.array(np.ones((2, 16), 'float32'), ctx=ctx(device))
        x.attach_grad()
        with autograd.record():
            loss = layer(x).sum()
        loss.backward()
        for pause in (False, True):
            with autograd.pause() if pause else autograd.predict_mode():
                q, s = mx.nd.RMSNorm(x, layer.gamma.data(), out_type='int8')
            assert (q.asnumpy() == 127).all()
            assert np.allclose(s.asnumpy(), 1 / 127)
    finally:
        set_native(prev)


@pytest.mark.parametrize('device', DEVICES)
def test_large_heads(native, device):
    """Refused at the call on the GPU, not where the result is read."""
    q = arr(np.random.RandomState(15).randn(1, 2, 136).astype('float32'),
            device)
    if device == 'gpu':
        with pytest.raises(ValueError):
            mx.nd.contrib.encdec_attention(q, q, q, heads=1)
    else:
        assert mx.nd.contrib.encdec_attention(q, q, q, heads=1).shape == q.shape
    assert mx.nd.contrib.encdec_attention(q, q, q, heads=2).shape == q.shape
