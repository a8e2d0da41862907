"""Sampling of tokens against the definition, one row at a time in 64 bits."""
import math

import numpy as np
import pytest
import torch

import mxnet_amd as mx

DEVICES = ['cpu', pytest.param('cuda:0', marks=pytest.mark.gpu)]
TYPES = [torch.float16, torch.bfloat16, torch.float32]
nd = mx.nd.from_torch


def oracle(x, u, temperature, top_k, top_p, min_p):
    """(token, log-probability, how near u is to a border of the tokens)"""
    x = np.where(np.isnan(x), -np.inf, x)
    order = np.lexsort((np.arange(len(x)), -x))
    top = x[order[0]]
    if top == -np.inf:
        return -1, math.nan, 1.0
    if not temperature > 0:
        return int(order[0]), 0.0, 1.0
    with np.errstate(invalid='ignore'):
        z = np.where(x[order] == top, 0.0, (x[order] - top) / temperature)
    w = np.exp(z)
    if top_k > 0:
        order, w = order[:top_k], w[:top_k]
    near = 1.0
    if top_p < 1:
        c = np.cumsum(w) / math.fsum(w)
        n = min(int((c < top_p).sum()) + 1, len(w))
        near = min(near, float(np.abs(c - top_p).min()))
        order, w = order[:n], w[:n]
    if min_p > 0:
        near = min(near, float(np.abs(w - min_p)[1:].min(initial=1.0)))
        n = max(1, int((w >= min_p).sum()))
        order, w = order[:n], w[:n]
    c = np.cumsum(w) / math.fsum(w)
    at = min(int((c <= u).sum()), len(w) - 1)
    near = min(near, float(np.abs(c - u)[:-1].min(initial=1.0)))
    return int(order[at]), math.log(w[at] / math.fsum(w)), near


def check(x, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    def row(p, i):
        return p[i].item() if isinstance(p, torch.Tensor) else p

    def arg(p):
        return nd(p) if isinstance(p, torch.Tensor) else p

    token, logp = mx.nd.contrib.sample_tokens(
        nd(x), nd(u), temperature=arg(temperature), top_k=arg(top_k),
        top_p=arg(top_p), min_p=arg(min_p), get_prob=True)
    token, logp = token.asnumpy(), logp.asnumpy()
    assert token.dtype == np.int32 and token.shape == (x.shape[0],)
    only = mx.nd.contrib.sample_tokens(
        nd(x), nd(u), temperature=arg(temperature), top_k=arg(top_k),
        top_p=arg(top_p), min_p=arg(min_p))
    assert np.array_equal(only.asnumpy(), token)
    rows = x.double().cpu().numpy()
    for i in range(len(rows)):
        want, lp, near = oracle(rows[i], float(u[i]), row(temperature, i),
                                row(top_k, i), row(top_p, i), row(min_p, i))
        if near < 1e-11:  # the oracle's own sums are not sure of it
            continue
        assert token[i] == want, (i, token[i], want, near)
        if want < 0:
            assert math.isnan(logp[i])
        else:
            # one rounding to float32, of a value whose parts are as large
            # as itself and the 64-bit sums' 1e-11
            assert abs(logp[i] - lp) <= abs(lp) * 2.0 ** -23 + 1e-9


def make(n, v, dtype, device, scale=2.5, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(n, v, generator=g) * scale).to(dtype).to(device)
    return x, torch.rand(n, generator=g).to(device)


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('n,v', [(1, 1), (3, 2), (5, 63), (2, 1001),
                                 (40, 4096), (1, 10000), (3, 30522),
                                 (130, 8193), (2, 70001)])
@pytest.mark.parametrize('kw', [
    {}, dict(temperature=0.7, top_k=50, top_p=0.9), dict(top_p=0.5),
    dict(top_k=1), dict(top_k=3, temperature=1.7), dict(min_p=0.05),
    dict(temperature=0.0), dict(top_p=0.0), dict(min_p=1.0),
    dict(temperature=1.3, top_k=1000, top_p=0.95, min_p=0.001)])
def test_against_definition(n, v, kw, dtype, device):
    x, u = make(n, v, dtype, device)
    check(x, u, **kw)


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('v', [5000, 60000])
def test_equal_and_flat_logits(v, dtype, device):
    """More equal or nearly equal logits than the kernel's list holds."""
    x, u = make(6, v, dtype, device, seed=1)
    x[0] = 1.5
    x[1] = (x[1] > 0).to(dtype)
    x[2] *= 1e-3
    x[3, ::2] = 7.0
    x[4] = torch.where(x[4] > 0, 0.0, -0.0).to(dtype)  # equal: 0 and -0
    for kw in ({}, dict(top_k=v // 3), dict(top_p=0.3), dict(min_p=0.5),
               dict(temperature=100.0, top_p=0.77, top_k=v - 1),
               dict(top_k=2500, top_p=0.9999)):
        check(x, u, **kw)


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('dtype', TYPES)
def test_masked_logits(dtype, device):
    """-inf, the lowest value, NaN and +inf in a row; rows without any."""
    x, u = make(8, 9000, dtype, device, seed=2)
    low = torch.finfo(dtype).min
    x[0, 10:] = -math.inf
    x[1, :8000] = low
    x[2, ::2] = math.nan
    x[3] = -math.inf
    x[4] = math.nan
    x[5, [7, 70, 700]] = math.inf
    x[6] = low
    x[7, 1:] = -math.inf
    for kw in ({}, dict(top_k=20, top_p=0.9), dict(min_p=0.1),
               dict(temperature=0.0), dict(top_k=5000)):
        check(x, u, **kw)


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('v', [700, 40000])
def test_parameters_by_row(v, device):
    x, u = make(6, v, torch.float32, device, seed=3)
    check(x, u,
          temperature=torch.tensor([0.0, 0.5, 1.0, 2.0, -1.0, 1.0],
                                   device=device),
          top_k=torch.tensor([0, 5, 0, 100, 7, -3], dtype=torch.int32,
                             device=device),
          top_p=torch.tensor([1.0, 0.9, 0.3, 0.8, 1.0, 2.0], device=device),
          min_p=torch.tensor([0.0, 0.0, 0.2, 0.01, 0.0, 0.0], device=device))


@pytest.mark.parametrize('device', DEVICES)
def test_numbers_at_their_ends(device):
    x, _ = make(5, 20000, torch.float32, device, seed=4)
    u = torch.tensor([0.0, 1 - 2.0 ** -24, 0.5, 2.0 ** -30, 1 - 2.0 ** -23],
                     device=device)
    for kw in ({}, dict(top_k=40), dict(top_p=0.9), dict(min_p=0.2)):
        check(x, u, **kw)
    # numbers outside of [0, 1) are taken to its ends
    out = torch.tensor([-1.0, 1.0, math.nan, math.inf, -math.inf],
                       device=device)
    ends = torch.tensor([0.0, 1 - 2.0 ** -24, 1 - 2.0 ** -24, 1 - 2.0 ** -24,
                         0.0], device=device)
    for kw in (dict(top_k=40), dict(top_p=0.9)):
        a = mx.nd.contrib.sample_tokens(nd(x), nd(out), **kw).asnumpy()
        b = mx.nd.contrib.sample_tokens(nd(x), nd(ends), **kw).asnumpy()
        assert np.array_equal(a, b)


@pytest.mark.parametrize('device', DEVICES)
def test_frequencies(device):
    """A uniform comb of numbers draws each token as often as its weight."""
    n = 4096
    x = torch.tensor([[0.0, 1.0, 2.0, -1.0]], device=device).repeat(n, 1)
    u = ((torch.arange(n, dtype=torch.float64) + 0.5) / n).float().to(device)
    t = mx.nd.contrib.sample_tokens(nd(x), nd(u), top_k=3).to_torch().cpu()
    p = torch.softmax(torch.tensor([0.0, 1.0, 2.0]), 0)
    got = torch.bincount(t.long(), minlength=4) / n
    assert float(got[3]) == 0
    assert float((got[:3] - p).abs().max()) < 2 / n


@pytest.mark.gpu
def test_views_streams_graphs():
    big = torch.randn(40, 20001, device='cuda:0')
    u = torch.rand(20, device='cuda:0')
    x = big[::2, 1:20000]
    check(x, u, top_p=0.9)
    check(x.half(), u, top_k=30)
    flat = torch.randn(3 * 9001 + 1, device='cuda:0').half()
    check(flat[1:].view(3, 9001), u[:3], temperature=0.5)
    kw = dict(top_p=0.8, temperature=0.9)
    want = mx.nd.contrib.sample_tokens(nd(x), nd(u), **kw).asnumpy()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = mx.nd.contrib.sample_tokens(nd(x), nd(u), **kw)
    side.synchronize()
    assert np.array_equal(got.asnumpy(), want)
    xs = [x.contiguous(), (x * 2).contiguous()]
    graphs, outs = [], []
    for v in xs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(mx.nd.contrib.sample_tokens(nd(v), nd(u), **kw))
        graphs.append(g)
    for k in range(3):
        u.uniform_()
        for v in xs:
            v.normal_()
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for v, o in zip(xs, outs):
            e = mx.nd.contrib.sample_tokens(nd(v), nd(u), **kw)
            assert np.array_equal(o.asnumpy(), e.asnumpy())


def test_refusals():
    f = mx.nd.contrib.sample_tokens
    x, u = torch.randn(2, 8), torch.rand(2)
    assert f(nd(x[:0]), nd(u[:0])).shape == (0,)
    for error, a, b, kw in [
            (TypeError, x.double(), u, {}), (ValueError, x[0], u, {}),
            (ValueError, x[:, :0], u, {}), (ValueError, x, u[:1], {}),
            (ValueError, x, u.double(), {}),
            (ValueError, x, u, dict(temperature=-1.0)),
            (ValueError, x, u, dict(temperature=math.nan)),
            (ValueError, x, u, dict(top_k=-1)),
            (ValueError, x, u, dict(top_k=1.5)),
            (ValueError, x, u, dict(top_p=1.5)),
            (ValueError, x, u, dict(min_p=-0.1)),
            (ValueError, x, u, dict(top_p=nd(torch.ones(3)))),
            (TypeError, x, u, dict(top_k=nd(torch.ones(2)))),
            (TypeError, x, u, dict(top_p=nd(torch.ones(2).int())))]:
        with pytest.raises(error):
            f(nd(a), nd(b), **kw)


@pytest.mark.parametrize('device', DEVICES)
def test_top_k_that_int32_does_not_hold(device):
    x, u = make(3, 50, torch.float32, device, seed=12)
    k = torch.tensor([(1 << 32) + 1, 1 << 31, 2], device=device)
    check(x, u, top_k=k)


@pytest.mark.gpu
def test_past_2_31_logits():
    """The last rows of 4 GB draw what they draw alone."""
    n, v = 8200, (1 << 18) + 8
    x = torch.empty(n, v, dtype=torch.float16, device='cuda:0')
    for i in range(0, n, 1000):
        x[i:i + 1000].normal_()
    u = torch.rand(n, device='cuda:0')
    last = x[-3:].clone()
    kw = dict(temperature=0.8, top_k=200, top_p=0.9, get_prob=True)
    token, logp = mx.nd.contrib.sample_tokens(nd(x), nd(u), **kw)
    alone = mx.nd.contrib.sample_tokens(nd(last), nd(u[-3:].clone()), **kw)
    assert torch.equal(token.to_torch()[-3:], alone[0].to_torch())
    assert torch.equal(logp.to_torch()[-3:], alone[1].to_torch())


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('dtype', TYPES)
def test_long_rows_in_parts(dtype, device):
    """Few rows of many logits, which the kernels count in parts."""
    x, u = make(4, 70001, dtype, device, seed=13)
    x[1, ::3] = -math.inf
    x[1, 69990:] = math.nan
    x[2] = math.nan
    x[3] = 0.25
    for kw in ({}, dict(top_k=60, top_p=0.9), dict(min_p=0.05),
               dict(temperature=0.0), dict(top_k=30000, top_p=0.7)):
        check(x, u, **kw)
    check(x, u, temperature=torch.tensor([0.5, 1, 2, 0], device=device),
          top_k=torch.tensor([0, 5, 0, 9], dtype=torch.int32, device=device))


@pytest.mark.gpu
def test_graphs_of_long_rows():
    """Two captured calls with workspaces, replayed in turn."""
    xs = [torch.randn(2, 80000, device='cuda:0') * 3 for _ in range(2)]
    u = torch.rand(2, device='cuda:0')
    kw = dict(top_p=0.8, top_k=1000, get_prob=True)
    graphs, outs = [], []
    for v in xs:
        mx.nd.contrib.sample_tokens(nd(v), nd(u), **kw)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(mx.nd.contrib.sample_tokens(nd(v), nd(u), **kw))
        graphs.append(g)
    for k in range(3):
        u.uniform_()
        for v in xs:
            v.normal_()
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for v, o in zip(xs, outs):
            e = mx.nd.contrib.sample_tokens(nd(v), nd(u), **kw)
            for a, b in zip(o, e):
                assert np.array_equal(a.asnumpy(), b.asnumpy())


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('v', [300, 70001])
@pytest.mark.parametrize('temperature', [5e-324, 1e-310, 1e-307, 1e-300])
def test_smallest_temperatures(temperature, v, device):
    """Whose reciprocal float64 does not hold: the largest logit, and one of
    those where several are equal."""
    x, u = make(4, v, torch.float32, device, seed=7)
    x[1, ::3] = 9.5
    x[2] = 0.0
    x[3, 5] = math.inf
    for kw in ({}, dict(top_k=7, top_p=0.5), dict(min_p=0.5)):
        check(x, u, temperature=temperature, **kw)
    rows = torch.tensor([1e-45, 1e-40, 1e-38, 0.0], device=device)
    check(x, u, temperature=rows)


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('v', [300, 70001])
def test_parameters_of_rows_outside_their_range(v, device):
    """Count as the nearest that lies in it, on the GPU as on the CPU."""
    x, u = make(6, v, torch.float32, device, seed=8)
    x[0, ::2] = -math.inf
    x[1, ::5] = math.inf
    x[2, ::3] = 9.5
    x[4, 1:] = -math.inf
    f = mx.nd.contrib.sample_tokens

    def rows(value, dtype=torch.float32):
        return nd(torch.full((6,), value, dtype=dtype, device=device))

    for name, value, near in (('temperature', math.inf, 1e30),
                              ('temperature', 3e38, 1e30),
                              ('temperature', -1.0, 0.0),
                              ('top_p', 1.5, 1.0), ('top_p', -1.0, 0.0),
                              ('min_p', 2.0, 1.0), ('min_p', -1.0, 0.0)):
        got = f(nd(x), nd(u), get_prob=True, **{name: rows(value)})
        want = f(nd(x), nd(u), get_prob=True, **{name: near})
        for g, w in zip(got, want):
            assert np.array_equal(g.asnumpy(), w.asnumpy()), (name, value)
        check(x, u, **{name: near})
    got = f(nd(x), nd(u), top_k=rows(-3, torch.int32))
    assert np.array_equal(got.asnumpy(), f(nd(x), nd(u)).asnumpy())
