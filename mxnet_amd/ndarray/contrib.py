"""Contrib operators: attention over an encoder's states, sampling of tokens,
and control flow.

Control-flow operators (reference src/operator/control_flow.cc:
``_foreach``, ``_while_loop``, ``_cond`` and python wrappers
python/mxnet/ndarray/contrib.py:foreach/while_loop/cond).

Imperative implementations over NDArray; autograd flows through the
underlying torch graph, so these are differentiable like the
reference's stateful control-flow ops.
"""
import torch

from .ndarray import NDArray
from ..ops import contrib_transformer as _ct
from ..ops import sampling as _sampling
from . import ops as _ops

__all__ = ['foreach', 'while_loop', 'cond', 'isinf', 'isnan', 'isfinite',
           'encdec_attention', 'sample_tokens']


def _as_list(x):
    return list(x) if isinstance(x, (list, tuple)) else [x]


def foreach(body, data, init_states):
    """Iterate ``body(step_data, states) -> (out, new_states)`` over the
    leading axis of ``data``; stacks per-step outputs
    (reference contrib.py:foreach / control_flow.cc ForeachOp)."""
    states = _as_list(init_states)
    data_list = _as_list(data)
    n = data_list[0].shape[0]
    outputs = []
    for i in range(n):
        step = [d[i] for d in data_list]
        out, states = body(step[0] if len(step) == 1 else step, states)
        outputs.append(_as_list(out))
    stacked = []
    for slot in zip(*outputs):
        stacked.append(NDArray(torch.stack([o.handle for o in slot])))
    out = stacked[0] if len(stacked) == 1 else stacked
    return out, states


def while_loop(cond_fn, func, loop_vars, max_iterations=None):
    """(reference contrib.py:while_loop): run ``func`` while ``cond_fn``
    holds; per-step outputs are stacked and padded to max_iterations."""
    loop_vars = _as_list(loop_vars)
    steps = 0
    outputs = []
    while bool(_scalar(cond_fn(*loop_vars))):
        if max_iterations is not None and steps >= max_iterations:
            break
        out, loop_vars = func(*loop_vars)
        loop_vars = _as_list(loop_vars)
        outputs.append(_as_list(out))
        steps += 1
    if not outputs:
        return [], loop_vars
    stacked = []
    for slot in zip(*outputs):
        st = torch.stack([o.handle for o in slot])
        if max_iterations is not None and steps < max_iterations:
            pad = torch.zeros((max_iterations - steps,) + tuple(st.shape[1:]),
                              dtype=st.dtype, device=st.device)
            st = torch.cat([st, pad])
        stacked.append(NDArray(st))
    out = stacked[0] if len(stacked) == 1 else stacked
    return out, loop_vars


def cond(pred, then_func, else_func):
    """(reference contrib.py:cond / CondOp)."""
    return then_func() if bool(_scalar(pred)) else else_func()


def _scalar(v):
    if isinstance(v, NDArray):
        return v.handle.item()
    if isinstance(v, torch.Tensor):
        return v.item()
    return v


def isinf(data):
    return NDArray(torch.isinf(data.handle))


def isnan(data):
    return NDArray(torch.isnan(data.handle))


def isfinite(data):
    return NDArray(torch.isfinite(data.handle))


def encdec_attention(queries, keys_values, values=None, heads=1,
                     kv_heads=None, valid_length=None, mask=None,
                     layout='NTC'):
    """Attention of a decoder's queries over an encoder's keys and values of
    another length, in one kernel; differentiable in all of them.

    queries (B, Sq, heads*D); keys_values (B, Sk, kv_heads*2*D) with each
    head's key before its value (the layout of interleaved_matmul_encdec_qk),
    or keys and ``values`` apart, (B, Sk, kv_heads*D) each; ``layout='TNC'``:
    time first.  Consecutive query heads share a key head where kv_heads is
    less than heads.  Keys from ``valid_length`` (B,) on and keys whose
    ``mask`` (B, Sk) is 0 are left out, whatever their memory holds; a row
    without a key gives zeros.  float16, bfloat16 and float32; head sizes up
    to 128 on the GPU.
    """
    if queries.is_native:
        return _encdec_native(queries, keys_values, values, heads, kv_heads,
                              valid_length, mask, layout)

    def t(x):
        return None if x is None else x._t
    return NDArray(_ct.encdec_attention(t(queries), t(keys_values), t(values),
                                        heads, kv_heads, t(valid_length),
                                        t(mask), layout))


def _encdec_native(queries, keys_values, values, heads, kv_heads,
                   valid_length, mask, layout):
    if layout not in ('NTC', 'TNC'):
        raise ValueError(f'encdec_attention: layout must be NTC or TNC, got '
                         f'{layout!r}')
    heads = int(heads)
    if heads > 0 and queries.shape[-1] // heads > 128 \
            and queries.context.device_type == 'gpu':
        raise ValueError(f'encdec_attention: head sizes up to 128 on the GPU, '
                         f'got {queries.shape[-1] // heads}')
    more = [values, valid_length, mask]
    attrs = {'heads': str(heads),
             'kv_heads': str(heads if kv_heads is None else int(kv_heads)),
             'tnc': '1' if layout == 'TNC' else '0'}
    for name, x in zip(('values', 'length', 'mask'), more):
        attrs['has_' + name] = '0' if x is None else '1'
    return _ops._ninv('_contrib_encdec_attention',
                      [queries, keys_values] + more, attrs, nout=2)[0]


def sample_tokens(logits, uniform, temperature=1.0, top_k=0, top_p=1.0,
                  min_p=0.0, get_prob=False):
    """The next token of each row of ``logits`` (N, V), drawn with the given
    random numbers ``uniform`` (N,) float32 in [0, 1).

    In the order of the logits, the largest first (of equal ones the lower
    index first), with weights exp((logit - max) / temperature): the first
    ``top_k`` are kept (0: all), of those the shortest prefix that holds
    ``top_p`` of their sum, of those the ones with at least ``min_p`` of the
    largest weight; the token is the first whose running sum exceeds uniform
    times the kept sum.  A temperature of 0 takes the largest logit.  Each
    parameter is a number, or an array of one for each row (float32, top_k
    int32), whose values count as the nearest of the parameter's range:
    temperature 0 to 1e30, top_k from 0 on, top_p and min_p 0 to 1.  A NaN is
    never drawn; a row without a finite or infinite logit gives -1.

    Returns int32 tokens (N,), or with ``get_prob`` ``[tokens, logp]``: the
    token's log-probability among the kept ones.  float16, bfloat16 and
    float32 logits, up to 2^19 a row; sums in 64 bits, the same at every call.
    """
    if logits.is_native:
        return _sample_native(logits, uniform, temperature, top_k, top_p,
                              min_p, get_prob)

    def t(x):
        return x._t if isinstance(x, NDArray) else x
    token, logp = _sampling.sample_tokens(
        logits._t, uniform._t, t(temperature), t(top_k), t(top_p), t(min_p),
        get_prob)
    return [NDArray(token), NDArray(logp)] if get_prob else NDArray(token)


def _sample_native(logits, uniform, temperature, top_k, top_p, min_p,
                   get_prob):
    ins, attrs = [logits, uniform], {}
    for name, value, dtype, low, high in (
            ('temperature', temperature, 'float32', 0.0, 1e30),
            ('top_k', top_k, 'int32', 0, (1 << 31) - 1),
            ('top_p', top_p, 'float32', 0.0, 1.0),
            ('min_p', min_p, 'float32', 0.0, 1.0)):
        if isinstance(value, NDArray):
            have = str(value.dtype)
            if ('float' in have) != ('float' in dtype):
                raise TypeError(f'sample_tokens: {name} of {have}')
            # (int64 as it is: int32 may not hold it)
            ins.append(value if have == dtype or have == 'int64'
                       else value.astype(dtype))
            attrs['has_' + name] = '1'
        else:
            attrs[name] = repr(_sampling.check_number(name, value, dtype, low,
                                                      high))
    token, logp = _ops._ninv('_contrib_sample_tokens', ins, attrs, nout=2)
    return [token, logp] if get_prob else token
