"""Operators of a decoder that reads an encoder: what is measured, on which
sizes, and the plain form that the kernels are compared with.

* ``norm``: ``mx.nd.RMSNorm`` with the residual's addition, forward and
  backward, and its int8 output with one scale a row;
* ``attention``: ``mx.nd.contrib.encdec_attention``, queries over an encoder's
  states of another length, forward and backward, and for single tokens;
* ``sample``: ``mx.nd.contrib.sample_tokens``, the next token from logits and
  given random numbers.
"""
import math

import numpy as np
import torch

own = False

DEV = 'cuda:0'
EPS = 1e-6
TYPES = {'float16': torch.float16, 'bfloat16': torch.bfloat16,
         'float32': torch.float32}


def listed():
    return [
        # one step of decoding for a batch of 32 sequences: latency
        dict(name='norm token', op='norm', mode='infer', rows=32, cols=1024,
             dtype='float16'),
        # one training step's norm at BERT-base width, 32 sequences of 128
        dict(name='norm train base', op='norm', mode='train', rows=4096,
             cols=768, dtype='float16'),
        # the norm before an int8 product, 64 sequences of 128
        dict(name='norm int8', op='norm', mode='int8', rows=8192, cols=1024,
             dtype='bfloat16'),
        # wide model, long batch
        dict(name='norm train wide', op='norm', mode='train', rows=16384,
             cols=4096, dtype='bfloat16'),
        # training at BERT-base width: targets of 64 over sources of 128
        dict(name='attention train base', op='attention', mode='train',
             batch=32, heads=12, kv_heads=12, dim=64, queries=64, keys=128,
             dtype='float16', masked=False, layout='NTC'),
        # long targets over long sources, heads as in BERT-large
        dict(name='attention train long', op='attention', mode='train',
             batch=4, heads=16, kv_heads=16, dim=64, queries=1024, keys=2048,
             dtype='bfloat16', masked=False, layout='NTC'),
        # ragged sizes, shared key heads, a key mask, time-major, fp32
        dict(name='attention ragged', op='attention', mode='infer', batch=7,
             heads=12, kv_heads=4, dim=64, queries=77, keys=509,
             dtype='float32', masked=True, layout='TNC'),
        # one token of 32 sequences over sources of BERT's longest length
        dict(name='attention token', op='attention', mode='infer', batch=32,
             heads=16, kv_heads=16, dim=64, queries=1, keys=512,
             dtype='float16', masked=False, layout='NTC'),
        # one token over a long document, shared key heads
        dict(name='attention token long', op='attention', mode='infer',
             batch=8, heads=32, kv_heads=8, dim=128, queries=1, keys=16384,
             dtype='bfloat16', masked=False, layout='NTC'),
        # one sequence of a word-level language model of 10000 words
        dict(name='sample one', op='sample', rows=1, vocab=10000,
             dtype='float32', temperature=0.8, top_k=0, top_p=0.95,
             min_p=0.0),
        # 32 sequences over BERT's vocabulary
        dict(name='sample batch', op='sample', rows=32, vocab=30522,
             dtype='float16', temperature=0.7, top_k=50, top_p=0.9,
             min_p=0.0),
        # many sequences over a large vocabulary
        dict(name='sample large', op='sample', rows=256, vocab=131072,
             dtype='bfloat16', temperature=1.0, top_k=0, top_p=0.95,
             min_p=0.02),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(['norm', 'attention', 'sample'])
    dtype = rng.choice(['float16', 'bfloat16', 'float32'])
    if op == 'norm':
        cols = _log(rng, 32, 8192)
        if rng.random() < 0.6:
            cols = max(8, cols // 8 * 8)
        most = max(1, min(32768, (1 << 25) // cols))
        return dict(op=op, mode=rng.choice(['infer', 'train', 'int8']),
                    rows=_log(rng, 1, most), cols=cols, dtype=dtype)
    if op == 'sample':
        vocab = _log(rng, 64, 131072)
        most = max(1, min(256, (1 << 24) // vocab))
        return dict(op=op, rows=_log(rng, 1, most), vocab=vocab, dtype=dtype,
                    temperature=rng.choice([0.5, 0.7, 1.0, 1.3]),
                    top_k=rng.choice([0, 0, 1, 20, 100, 1000]),
                    top_p=rng.choice([1.0, 0.95, 0.8, 0.5]),
                    min_p=rng.choice([0.0, 0.0, 0.05]))
    kv_heads = rng.choice([1, 2, 4, 8, 12, 16])
    heads = kv_heads * rng.choice([1, 1, 2, 4])
    dim = rng.choice([16, 32, 40, 64, 64, 80, 128])
    mode = rng.choice(['train', 'infer', 'token'])
    queries = 1 if mode == 'token' else _log(rng, 2, 1024)
    keys = _log(rng, 1, 16384 if mode == 'token' else 2048)
    # fp32 goes at the matrix cores' fp32 rate: smaller ones of it
    most = (1 << 32) if dtype != 'float32' else (1 << 29)
    queries = max(1, min(queries, most // (heads * dim * keys)))
    batch = max(1, min(32, most // (heads * dim * keys * queries),
                       (1 << 25) // (kv_heads * dim * keys)))
    return dict(op=op, mode='train' if mode == 'train' else 'infer',
                batch=rng.randint(1, batch), heads=heads, kv_heads=kv_heads,
                dim=dim, queries=queries, keys=keys, dtype=dtype,
                masked=rng.random() < 0.5,
                layout=rng.choice(['NTC', 'TNC']))


def _lengths(case):
    """One length for each sequence of the batch, evenly from half to full:
    the seed only decides which sequence has which, so the work is the
    case's alone."""
    b, k = case['batch'], case['keys']
    if b == 1:
        return [k]
    return [k - (k // 2) * i // (b - 1) for i in range(b)]


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    t = TYPES[case['dtype']]

    def normal(*shape, scale=1.0, dtype=t):
        return (torch.randn(*shape, generator=g, device=DEV) * scale).to(dtype)

    s = {'case': case}
    if case['op'] == 'norm':
        r, c = case['rows'], case['cols']
        s['x'] = normal(r, c)
        s['residual'] = normal(r, c, scale=2.0)
        s['gamma'] = 1.0 + normal(c, scale=0.2, dtype=torch.float32)
        if case['mode'] == 'train':
            s['dy'] = normal(r, c)
            s['dsum'] = normal(r, c)
        return s
    if case['op'] == 'sample':
        # logits as a trained model's: a few likely tokens, a long tail
        x = torch.randn(case['rows'], case['vocab'], generator=g, device=DEV)
        s['logits'] = (2.5 * x).to(t)
        s['uniform'] = torch.rand(case['rows'], generator=g, device=DEV)
        return s
    b, h, hk, d = (case[k] for k in ('batch', 'heads', 'kv_heads', 'dim'))
    nq, nk = case['queries'], case['keys']

    def lead(n):
        return (b, n) if case['layout'] == 'NTC' else (n, b)

    s['queries'] = normal(*lead(nq), h * d)
    s['keys_values'] = normal(*lead(nk), hk * 2 * d)
    order = np.random.RandomState(seed % (1 << 32)).permutation(b)
    s['lengths'] = torch.tensor([_lengths(case)[i] for i in order],
                                dtype=torch.int32, device=DEV)
    s['mask'] = None
    if case['masked']:
        s['mask'] = torch.rand(b, nk, generator=g, device=DEV) < 0.9
    if case['mode'] == 'train':
        s['dout'] = normal(*lead(nq), h * d)
    return s


# -- plain forms ------------------------------------------------------------

def _norm_plain(s):
    x, mode = s['x'], s['case']['mode']
    h = (x.float() + s['residual'].float()).to(x.dtype)
    hf = h.float()
    # the mean of the squares in 64 bits: an int8 step lies next to a border
    r = (1.0 / torch.sqrt(hf.double().square().mean(-1, keepdim=True)
                          + EPS)).float()
    y = hf * r * s['gamma']
    if mode == 'infer':
        return y.to(x.dtype), h
    if mode == 'int8':
        top = y.abs().amax(-1, keepdim=True)
        scale = torch.where(top > 0, top / 127.0, torch.ones_like(top))
        q = torch.round(y * torch.where(top > 0, 127.0 / top,
                                        torch.zeros_like(top)))
        return q.clamp(-127, 127).to(torch.int8) * scale, h
    dy = s['dy'].float()
    g = dy * s['gamma']
    n = hf * r
    dh = r * (g - n * (g * n).mean(-1, keepdim=True)) + s['dsum'].float()
    return (y.to(x.dtype), h, dh.to(x.dtype), (dy * n).sum(0))


def _heads_first(t, layout, n, d):
    """[B,S,n*d] or [S,B,n*d] to [B,n,S,d] in 32 bits."""
    t = t.float().reshape(t.shape[0], t.shape[1], n, d)
    return t.permute(*((0, 2, 1, 3) if layout == 'NTC' else (1, 2, 0, 3))) \
        .contiguous()


def _heads_last(t, layout):
    b, n, s, d = t.shape
    return t.permute(*((0, 2, 1, 3) if layout == 'NTC' else (2, 0, 1, 3))) \
        .reshape(*((b, s) if layout == 'NTC' else (s, b)), n * d)


def _attention_plain(s):
    c = s['case']
    h, hk, d, layout = c['heads'], c['kv_heads'], c['dim'], c['layout']
    b, nq, nk, t = c['batch'], c['queries'], c['keys'], s['queries'].dtype
    scale = 1.0 / math.sqrt(d)
    q = _heads_first(s['queries'], layout, h, d).reshape(b, hk, -1, d)
    kv = _heads_first(s['keys_values'], layout, hk, 2 * d)
    k, v = kv[..., :d].contiguous(), kv[..., d:].contiguous()
    keep = torch.arange(nk, device=DEV)[None] < s['lengths'][:, None]
    if s['mask'] is not None:
        keep = keep & s['mask']
    keep = keep[:, None, None]
    x = torch.matmul(q, k.transpose(-1, -2).contiguous()) * scale
    x = x.masked_fill(~keep, float('-inf'))
    top = x.amax(-1, keepdim=True)
    p = torch.exp(x - torch.where(top == float('-inf'),
                                  torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total == 0, torch.ones_like(total), total)
    o = torch.matmul(p, v)
    out = _heads_last(o.reshape(b, h, nq, d), layout).to(t)
    if c['mode'] == 'infer':
        return out
    do = _heads_first(s['dout'], layout, h, d).reshape(b, hk, -1, d)
    dv = torch.matmul(p.transpose(-1, -2).contiguous(), do)
    dp = torch.matmul(do, v.transpose(-1, -2).contiguous())
    ds = p * (dp - (do * o).sum(-1, keepdim=True)) * scale
    dq = torch.matmul(ds, k)
    dk = torch.matmul(ds.transpose(-1, -2).contiguous(), q)
    return (out, _heads_last(dq.reshape(b, h, nq, d), layout).to(t),
            _heads_last(torch.cat([dk, dv], -1), layout).to(t))


def _sample_plain(s):
    c = s['case']
    x, order = torch.sort(s['logits'].float(), dim=-1, descending=True,
                          stable=True)
    # in 64 bits: whether a token is kept or drawn lies next to a border
    w = torch.exp((x.double() - x[:, :1].double()) / c['temperature'])
    if 0 < c['top_k'] < c['vocab']:
        w[:, c['top_k']:] = 0
    if c['top_p'] < 1.0:
        cum = torch.cumsum(w, -1)
        w = w.masked_fill(cum - w >= c['top_p'] * cum[:, -1:], 0.0)
    if c['min_p'] > 0:
        w = w.masked_fill(w < c['min_p'], 0.0)
    cum = torch.cumsum(w, -1)
    total = cum[:, -1:]
    at = (cum <= s['uniform'].double()[:, None] * total).sum(-1, keepdim=True)
    token = order.gather(1, at)[:, 0].to(torch.int32)
    return token, torch.log(w.gather(1, at) / total)[:, 0].float()


# -- the framework's operators ----------------------------------------------

def _norm_own(s):
    import mxnet_amd as mx
    nd, mode = mx.nd.from_torch, s['case']['mode']
    if mode == 'train':
        x = nd(s['x'].detach().requires_grad_())
        res = nd(s['residual'])
        gamma = nd(s['gamma'].detach().requires_grad_())
        with mx.autograd.record():
            y, h = mx.nd.RMSNorm(x, gamma, residual=res, eps=EPS)
        dx, dgamma = mx.autograd.grad([y, h], [x, gamma],
                                      [nd(s['dy']), nd(s['dsum'])])
        return (y.to_torch().detach(), h.to_torch().detach(), dx.to_torch(),
                dgamma.to_torch())
    args = (nd(s['x']), nd(s['gamma']))
    if mode == 'infer':
        y, h = mx.nd.RMSNorm(*args, residual=nd(s['residual']), eps=EPS)
        return y.to_torch(), h.to_torch()
    q, scale, h = mx.nd.RMSNorm(*args, residual=nd(s['residual']), eps=EPS,
                                out_type='int8')
    return q.to_torch() * scale.to_torch(), h.to_torch()


def _attention_own(s):
    import mxnet_amd as mx
    c, nd = s['case'], mx.nd.from_torch
    kw = dict(heads=c['heads'], kv_heads=c['kv_heads'], layout=c['layout'],
              valid_length=nd(s['lengths']),
              mask=None if s['mask'] is None else nd(s['mask']))
    if c['mode'] == 'infer':
        return mx.nd.contrib.encdec_attention(
            nd(s['queries']), nd(s['keys_values']), **kw).to_torch()
    q = nd(s['queries'].detach().requires_grad_())
    kv = nd(s['keys_values'].detach().requires_grad_())
    with mx.autograd.record():
        out = mx.nd.contrib.encdec_attention(q, kv, **kw)
    dq, dkv = mx.autograd.grad([out], [q, kv], [nd(s['dout'])])
    return out.to_torch().detach(), dq.to_torch(), dkv.to_torch()


def _sample_own(s):
    import mxnet_amd as mx
    c, nd = s['case'], mx.nd.from_torch
    token, logp = mx.nd.contrib.sample_tokens(
        nd(s['logits']), nd(s['uniform']), temperature=c['temperature'],
        top_k=c['top_k'], top_p=c['top_p'], min_p=c['min_p'], get_prob=True)
    return token.to_torch(), logp.to_torch()


def run(state):
    op = state['case']['op']
    if own:
        return {'norm': _norm_own, 'attention': _attention_own,
                'sample': _sample_own}[op](state)
    return {'norm': _norm_plain, 'attention': _attention_plain,
            'sample': _sample_plain}[op](state)


def work(case):
    size = 4 if case['dtype'] == 'float32' else 2
    if case['op'] == 'norm':
        r, c, mode = case['rows'], case['cols'], case['mode']
        # in: data, residual; out: norm (or int8, its scale and the values
        # it stands for), sum; backward: two gradients in, one out
        n = r * c
        if mode == 'infer':
            return {'bytes': 4 * n * size + 4 * c, 'flops': 5 * n}
        if mode == 'int8':
            return {'bytes': 3 * n * size + n + 4 * n + 4 * r + 4 * c,
                    'flops': 8 * n}
        return {'bytes': 7 * n * size + 8 * c, 'flops': 16 * n}
    if case['op'] == 'sample':
        n = case['rows'] * case['vocab']
        return {'bytes': n * size + 12 * case['rows'], 'flops': 4 * n}
    h, hk, d, b, nq = (case[k] for k in ('heads', 'kv_heads', 'dim', 'batch',
                                         'queries'))
    keys = sum(_lengths(case))
    q = b * nq * h * d * size
    kv = keys * hk * 2 * d * size
    flops = 4 * h * nq * keys * d
    if case['mode'] == 'infer':
        return {'bytes': 2 * q + kv, 'flops': flops}
    # backward: five products to the forward's two; the whole gradient of the
    # keys and values is written, zeros at masked places among it
    dkv = b * case['keys'] * hk * 2 * d * size
    return {'bytes': 4 * q + kv + dkv, 'flops': flops * 7 // 2}


# -- the definitions in 64 bits ---------------------------------------------

def _norm_exact(s):
    f64 = torch.float64
    h = (s['x'].to(f64) + s['residual'].to(f64)).to(s['x'].dtype)
    v, gamma = h.to(f64), s['gamma'].to(f64)
    c = v.shape[-1]
    # the sum is rounded to its type, where it is stored, before the norm
    ms = torch.einsum('rc,rc->r', v, v)[:, None] / c + EPS
    n = v / torch.sqrt(ms)
    y = n * gamma
    mode = s['case']['mode']
    if mode == 'infer':
        return y, v
    if mode == 'int8':
        return None, v
    dy, dsum = s['dy'].to(f64), s['dsum'].to(f64)
    g = dy * gamma
    dot = torch.einsum('rc,rc->r', g, v)[:, None]
    dh = g / torch.sqrt(ms) - v * dot / (c * ms * torch.sqrt(ms)) + dsum
    return y, v, dh, torch.einsum('rc,rc->c', dy, n)


def _attention_exact(s):
    """One sequence and one shared head at a time, over its valid keys."""
    c, f64 = s['case'], torch.float64
    h, hk, d = c['heads'], c['kv_heads'], c['dim']
    grp = h // hk
    rows = (lambda t: t) if c['layout'] == 'NTC' else \
        (lambda t: t.transpose(0, 1))
    q, kv = rows(s['queries']), rows(s['keys_values'])
    train = c['mode'] == 'train'
    out = torch.zeros(q.shape, dtype=f64, device=DEV)
    dq, dkv = torch.zeros_like(out), torch.zeros(kv.shape, dtype=f64,
                                                 device=DEV)
    for b in range(c['batch']):
        idx = torch.arange(int(s['lengths'][b]), device=DEV)
        if s['mask'] is not None:
            idx = idx[s['mask'][b, :len(idx)]]
        if not len(idx):
            continue
        for j in range(hk):
            k = kv[b, idx, 2 * d * j:2 * d * j + d].to(f64)
            v = kv[b, idx, 2 * d * j + d:2 * d * (j + 1)].to(f64)
            cols = slice(j * grp * d, (j + 1) * grp * d)
            qq = q[b, :, cols].to(f64).reshape(-1, d)
            z = qq @ k.T / math.sqrt(d)
            p = torch.exp(z - torch.logsumexp(z, -1, keepdim=True))
            o = p @ v
            out[b, :, cols] = o.reshape(-1, grp * d)
            if train:
                do = rows(s['dout'])[b, :, cols].to(f64).reshape(-1, d)
                dp = do @ v.T
                ds = p * (dp - (p * dp).sum(-1, keepdim=True)) / math.sqrt(d)
                dq[b, :, cols] = (ds @ k).reshape(-1, grp * d)
                dkv[b, idx, 2 * d * j:2 * d * j + d] = ds.T @ qq
                dkv[b, idx, 2 * d * j + d:2 * d * (j + 1)] = p.T @ do
    out, dq, dkv = rows(out), rows(dq), rows(dkv)
    return (out, dq, dkv) if train else out


def _sample_exact(s):
    c = s['case']
    if c['rows'] * c['vocab'] > 1 << 22:
        return None
    logits = s['logits'].double().cpu().numpy()
    uniform = s['uniform'].double().cpu().numpy()
    tokens, logps = [], []
    for x, u in zip(logits, uniform):
        order = np.lexsort((np.arange(len(x)), -x))
        if c['top_k'] > 0:
            order = order[:c['top_k']]
        p = np.exp((x[order] - x[order[0]]) / c['temperature'])
        p /= math.fsum(p)
        n = len(p)
        if c['top_p'] < 1.0:
            n = min(n, int(np.searchsorted(np.cumsum(p), c['top_p'])) + 1)
        if c['min_p'] > 0:
            n = min(n, int((p >= c['min_p'] * p[0]).sum()))
        p = p[:n] / math.fsum(p[:n])
        at = min(int(np.searchsorted(np.cumsum(p), u, side='right')), n - 1)
        tokens.append(int(order[at]))
        logps.append(math.log(p[at]))
    return np.array(tokens, np.int32), np.array(logps)


def exact(case, seed):
    s = prepare(case, seed)
    return {'norm': _norm_exact, 'attention': _attention_exact,
            'sample': _sample_exact}[case['op']](s)
