"""encdec_attention and sample_tokens in hybrid_forward, as graph nodes, and
under mx.npx."""
import numpy as np
import pytest

import mxnet_amd as mx
from mxnet_amd.base import set_native
from mxnet_amd.gluon import SymbolBlock, nn

DEVICES = ['cpu', pytest.param('gpu', marks=pytest.mark.gpu)]


def ctx(device):
    return mx.cpu() if device == 'cpu' else mx.gpu(0)


class Block(nn.HybridBlock):
    """Attention of a layer's own states, in the classic protocol."""

    def __init__(self, **kw):
        super().__init__(**kw)
        self.query = nn.Dense(32, flatten=False, in_units=32)
        self.key_value = nn.Dense(32, flatten=False, in_units=32)
        self.norm = nn.RMSNorm()

    def hybrid_forward(self, F, x):
        a = F.contrib.encdec_attention(self.query(x), self.key_value(x),
                                       heads=4, kv_heads=2)
        return self.norm(a, x)[0]


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('native', [False, True])
def test_in_hybrid_forward_and_exported(native, device, tmp_path):
    prev = set_native(native)
    try:
        net = Block()
        net.initialize(ctx=ctx(device))
        rs = np.random.RandomState(0)
        x = mx.nd.array(rs.randn(2, 5, 32).astype('float32'), ctx=ctx(device))
        want = net(x).asnumpy()
        q, kv = net.query(x), net.key_value(x)
        a = mx.nd.contrib.encdec_attention(q, kv, heads=4, kv_heads=2)
        assert np.array_equal(net.norm(a, x)[0].asnumpy(), want)
        files = net.export(str(tmp_path / 'net'))
        again = SymbolBlock.imports(files[0], ['data'], files[1],
                                    ctx=ctx(device))
        assert np.array_equal(again(x).asnumpy(), want)
        net.hybridize()
        for _ in range(3):
            assert np.array_equal(net(x).asnumpy(), want)
    finally:
        set_native(prev)


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('native', [False, True])
def test_nodes_with_every_argument(native, device, tmp_path):
    prev = set_native(native)
    try:
        rs = np.random.RandomState(1)

        def a(v):
            return mx.nd.array(v, ctx=ctx(device), dtype=str(v.dtype))

        feed = dict(q=rs.randn(5, 3, 16), k=rs.randn(7, 3, 8),
                    v=rs.randn(7, 3, 8), x=rs.randn(3, 50))
        feed = {k: a(v.astype('float32')) for k, v in feed.items()}
        feed['n'] = a(np.array([7, 0, 3], 'int64'))
        feed['m'] = a((rs.rand(3, 7) < 0.6).astype('uint8'))
        feed['u'] = a(rs.rand(3).astype('float32'))
        feed['t'] = a(np.array([0.5, 0, 2], 'float32'))
        s = {k: mx.sym.var(k) for k in feed}
        out = mx.sym.contrib.encdec_attention(
            s['q'], s['k'], s['v'], heads=4, kv_heads=2, layout='TNC',
            valid_length=s['n'], mask=s['m'])
        token, logp = mx.sym.contrib.sample_tokens(
            s['x'], s['u'], temperature=s['t'], top_k=20, top_p=0.9,
            min_p=0.01, get_prob=True)
        only = mx.sym.contrib.sample_tokens(s['x'], s['u'])
        net = mx.sym.Group([out, token, logp, only])
        net.save(str(tmp_path / 'n.json'))
        want = [mx.nd.contrib.encdec_attention(
            feed['q'], feed['k'], feed['v'], heads=4, kv_heads=2,
            layout='TNC', valid_length=feed['n'], mask=feed['m'])]
        want += mx.nd.contrib.sample_tokens(
            feed['x'], feed['u'], temperature=feed['t'], top_k=20, top_p=0.9,
            min_p=0.01, get_prob=True)
        want += [mx.nd.contrib.sample_tokens(feed['x'], feed['u'])]
        for g in (net, mx.sym.load(str(tmp_path / 'n.json'))):
            got = g.eval_dict(feed)
            assert len(got) == len(want)
            for b, w in zip(got, want):
                assert np.array_equal(b.asnumpy(), w.asnumpy())
        assert np.array_equal(
            mx.npx.sample_tokens(feed['x'], feed['u']).asnumpy(),
            want[3].asnumpy())
        assert np.array_equal(mx.npx.encdec_attention(
            feed['q'], feed['k'], feed['v'], heads=4, kv_heads=2,
            layout='TNC', valid_length=feed['n'],
            mask=feed['m']).asnumpy(), want[0].asnumpy())
    finally:
        set_native(prev)


def test_saved_again_after_loading():
    """A loaded graph knows how many outputs its nodes have."""
    x, r, g = (mx.sym.var(n) for n in 'xrg')
    y, h = mx.sym.RMSNorm(x, g, residual=r)
    token, logp = mx.sym.contrib.sample_tokens(y, h, get_prob=True)
    net = mx.sym.Group([y, h, token, logp])
    again = mx.sym.load_json(net.tojson())
    assert again.tojson() == net.tojson()
    assert again[1].tojson() == logp.tojson()
