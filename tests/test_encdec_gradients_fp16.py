"""Gradients of the attention in fp16 where dS lies outside of what fp16 holds
in full: small and large output gradients, long rows.  A kernel that rounds P
and dS as they are loses them below 2^-14 and over 2^16."""
import math

import pytest
import torch

from test_encdec_attention import U32, call, make

HALF = 2.0 ** -25  # half a step of fp16 below its normal numbers
u = 2.0 ** -11


def exact(d, size, most=15):
    """Gradients in 64 bits, and how far rounding may take a kernel from them
    that takes P and dS times the power of two that brings the largest dS to
    2^13 or more, or times 2^most where it stays below that."""
    B, H, Hk, sq, sk, D = size
    G = H // Hk

    def split(t, n, w):
        return t.double().reshape(B, -1, n, w).transpose(1, 2)

    kv = split(d['kv'], Hk, 2 * D)
    k, v = (t.repeat_interleave(G, 1) for t in (kv[..., :D], kv[..., D:]))
    q, do = split(d['q'], H, D), split(d['dout'], H, D)
    c = 1 / math.sqrt(D)
    s = q @ k.transpose(-1, -2).contiguous() * c
    p = torch.softmax(s, -1)
    o = p @ v
    ka, va, qa, ga = k.abs(), v.abs(), q.abs(), do.abs()
    # scores are sums of D products in 32 bits, their log-sum of sk weights;
    # the shift goes into the log-sum with one more step of it
    score = (qa @ ka.transpose(-1, -2).contiguous()).amax(-1, keepdim=True) * c
    lse = torch.logsumexp(s, -1, keepdim=True).abs() + 15
    e = 2 * (D + 4) * U32 * score + 6 * U32 * lse + (64 + sk) * U32
    dp = do @ v.transpose(-1, -2).contiguous()
    w = p * (dp - (do * o).sum(-1, keepdim=True))
    # the power of two, at least: half a step below fp16's normal numbers is
    # that much smaller for P and dS.  (One over 2^13 for the largest dS goes
    # to V, which then has half steps of its own.)
    down = float(w.abs().max()) * 2.0 ** -12
    of_ds = HALF * max(2.0 ** -most, down)
    of_p = HALF * max(2.0 ** -most, min(1.0, down))
    of_v = HALF * down if down > 1 else 0.0
    o_off = (p @ va) * (u + e) + u * o.abs() + HALF * (
        1 + va.sum(2, keepdim=True))
    w_off = w.abs() * (u + e) + of_ds + p * (
        (D + 4) * U32 * (ga @ va.transpose(-1, -2).contiguous())
        + (ga * (o_off + D * U32 * o.abs() + of_v)).sum(-1, keepdim=True))
    n = sk * U32
    dq, dq_off = w @ k * c, (w_off + n * w.abs()) @ ka * c
    n = sq * G * U32
    wt, pt = (t.transpose(-1, -2).contiguous() for t in (w, p))
    dk, dv = wt @ q * c, pt @ do
    dk_off = (w_off + n * w.abs()).transpose(-1, -2).contiguous() @ qa * c
    dv_off = pt @ (ga * (u + e + n)) + of_p * ga.sum(2, keepdim=True)

    def join(t):
        return t.transpose(1, 2).reshape(B, t.shape[2], -1)

    def shared(t):
        return t.reshape(B, Hk, G, sk, D).sum(2)

    pairs = [(dq, dq_off), (torch.cat([shared(dk), shared(dv)], -1),
                            torch.cat([shared(dk_off), shared(dv_off)], -1))]
    # each result is rounded to fp16 at the end
    return [(join(a), join(b * (1 + u) + a.abs() * u * 1.01 + HALF))
            for a, b in pairs]


def compare(d, size, most=15):
    got = call(d, size, 'NTC', grad=True)[1:]
    for name, g, (w, off) in zip(('dq', 'dkv'), got, exact(d, size, most)):
        assert float(w.abs().max()) < 65504
        ratio = ((g.double() - w).abs() / off).max()
        assert ratio <= 1, (name, float(ratio), float(w.abs().max()))


SIZES = [(1, 2, 2, 1024, 2048, 64), (2, 4, 2, 70, 300, 32),
         (1, 2, 1, 200, 500, 96), (1, 2, 2, 130, 1000, 128),
         (1, 8, 8, 1, 3000, 64), (1, 1, 1, 40, 20000, 32),
         (1, 4, 2, 9, 3000, 40), (1, 3, 1, 333, 77, 5)]


@pytest.mark.gpu
@pytest.mark.parametrize('size', SIZES)
@pytest.mark.parametrize('power', [0, -7, -10, -13, -17, -20])
def test_small_gradients(power, size):
    d = make(size, torch.float32, 'cuda:0', seed=31)
    d['dout'] *= 2.0 ** power
    d = {k: v.half() if v is not None else v for k, v in d.items()}
    compare(d, size)


@pytest.mark.gpu
@pytest.mark.parametrize('size', SIZES)
@pytest.mark.parametrize('power,of_v', [(6, 0), (12, 0), (12, 6), (12, 10)])
def test_large_gradients(power, of_v, size):
    """dS up to 2^20 and more, and small queries and keys, so that the
    gradients themselves are numbers of fp16."""
    d = make(size, torch.float32, 'cuda:0', seed=32)
    D = size[5]
    # (no further: what counts is dS)
    d['dout'] = (d['dout'] * 2.0 ** power / max(1, size[3] // 64)).clamp(
        -30000, 30000)
    low = 2.0 ** -(max(0, power + of_v - 6))
    kv = d['kv'].view(size[0], size[4], size[2], 2, D)
    kv[:, :, :, 0] *= low
    kv[:, :, :, 1] *= 2.0 ** of_v
    d['q'] *= low
    d = {k: v.half() if v is not None else v for k, v in d.items()}
    compare(d, size)


@pytest.mark.gpu
@pytest.mark.parametrize('size', [(1, 2, 2, 100, 200, 64),
                                  (1, 8, 2, 3, 3000, 32)])
def test_rows_of_every_size_of_gradient(size):
    """A row's dQ does not lose bits to other rows' gradients."""
    d = make(size, torch.float32, 'cuda:0', seed=33)
    rows = torch.arange(size[3], device='cuda:0')
    factor = 2.0 ** (10 - (rows * 5) % 23).float()
    d['dout'] *= factor[None, :, None]
    d = {k: v.half() if v is not None else v for k, v in d.items()}
    got = call(d, size, 'NTC', grad=True)[1]
    for at in range(0, size[3], 7):
        one = dict(d, dout=torch.zeros_like(d['dout']))
        one['dout'][:, at] = d['dout'][:, at]
        w, off = exact(one, size)[0]
        assert ((got.double() - w).abs() <= off)[:, at].all()


@pytest.mark.gpu
@pytest.mark.parametrize('bad', [math.inf, math.nan])
def test_an_infinite_gradient_of_one_row(bad):
    """Reaches every key's column of dV that it lies in and no other, and no
    other row's dQ (which were finite before P and dS had a factor)."""
    size = (1, 2, 2, 70, 90, 64)
    d = make(size, torch.float16, 'cuda:0', seed=34)
    d['dout'] = d['dout'] * 2.0 ** -6  # no row lowers the shift
    want = call(d, size, 'NTC', grad=True)[1:]
    d['dout'] = d['dout'].clone()
    d['dout'][0, 13, 64 + 5] = bad  # the second head's sixth column
    dq, dkv = call(d, size, 'NTC', grad=True)[1:]
    rows = torch.arange(70, device='cuda:0') != 13
    assert torch.equal(dq[:, rows], want[0][:, rows])
    assert torch.equal(dq[..., :64], want[0][..., :64])
    assert not torch.isfinite(dq[0, 13, 64:]).any()
    kv = dkv.view(90, 2, 2, 64)
    assert torch.equal(kv[:, 0], want[1].view(90, 2, 2, 64)[:, 0])
    assert not torch.isfinite(kv[:, 1, 1, 5]).any()
    assert not torch.isfinite(kv[:, 1, 0]).any()
    others = torch.arange(64, device='cuda:0') != 5
    assert torch.equal(kv[:, 1, 1][:, others],
                       want[1].view(90, 2, 2, 64)[:, 1, 1][:, others])


@pytest.mark.gpu
@pytest.mark.parametrize('power,times', [(-10, 512), (0, 512), (8, 512),
                                         (-10, 16384), (0, 16384)])
def test_large_scores(power, times):
    """Log-sums of 2^17, and of every third row over 2^20, which takes no
    shift (whose weights float32 does not hold to more than a few bits)."""
    size = (1, 2, 1, 66, 96, 16)
    g = torch.Generator().manual_seed(35)
    d = make(size, torch.float16, 'cuda:0', seed=35)
    q = torch.randint(-3, 4, (1, 66, 32), generator=g).half()
    q[:, ::3] *= times
    d['q'] = q.to('cuda:0')
    d['kv'][:, :, :16] = 16 * torch.randint(-3, 4, (1, 96, 16),
                                            generator=g).to('cuda:0')
    d['dout'] = d['dout'] * 2.0 ** power
    s = q[0, :, :16].double() @ d['kv'][0, :, :16].double().cpu().T
    over = 2.0 ** (16 if times == 512 else 20)
    assert int((s.amax(1) / 4 * 1.4427 > over).sum()) > 5
    # a row without a shift leaves its head's P and dS none: they have fp16's
    # own half steps below its normal numbers
    compare(d, size, 15 if times == 512 else 0)
