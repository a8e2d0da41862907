"""Sampling of tokens from logits with given random numbers.

GPU: the kernels of src/ops/sample.hip.  CPU: the formula in 64 bits, the
numerics oracle.
"""
import math

import torch

from .dispatch import hip_required, use_hip

__all__ = ['sample_tokens']


def _param(name, value, n, device, dtype, low, high):
    """A checked number, or a tensor of one a row."""
    if isinstance(value, torch.Tensor):
        if value.shape != (n,):
            raise ValueError(f'sample_tokens: {name} must be one number or '
                             f'one for each of {n} rows, got '
                             f'{tuple(value.shape)}')
        if value.device != device:
            raise ValueError(f'sample_tokens: logits on {device}, {name} on '
                             f'{value.device}')
        if value.is_floating_point() != dtype.is_floating_point:
            raise TypeError(f'sample_tokens: {name} of {value.dtype}')
        if value.dtype == torch.int64:  # int32 may not hold it
            value = value.clamp(0, high)
        return value.to(dtype).contiguous()
    return check_number(name, value, str(dtype).replace('torch.', ''), low,
                        high)


def check_number(name, value, dtype, low, high):
    """A parameter that is one number: its value, if it lies in its range."""
    if dtype == 'int32':
        if int(value) != value:
            raise ValueError(f'sample_tokens: {name} must be a whole number, '
                             f'got {value!r}')
        value = int(value)
    else:
        value = float(value)
    if not low <= value <= high:
        raise ValueError(f'sample_tokens: {name} must lie in {low} to {high}, '
                         f'got {value!r}')
    return value


def sample_tokens(logits, uniform, temperature=1.0, top_k=0, top_p=1.0,
                  min_p=0.0, get_prob=False):
    """See mx.nd.contrib.sample_tokens.  Returns (tokens, log-probabilities
    or None)."""
    if logits.dtype not in (torch.float16, torch.bfloat16, torch.float32):
        raise TypeError(f'sample_tokens: float16, bfloat16 or float32 logits, '
                        f'got {logits.dtype}')
    if logits.dim() != 2 or not 1 <= logits.shape[1] <= 1 << 19:
        raise ValueError(f'sample_tokens: rows of 1 to {1 << 19} logits, got '
                         f'{tuple(logits.shape)}')
    n, dev = logits.shape[0], logits.device
    if n >= 1 << 20:
        raise ValueError(f'sample_tokens: less than {1 << 20} rows, got {n}')
    if uniform.shape != (n,) or uniform.dtype != torch.float32 \
            or uniform.device != dev:
        raise ValueError(f'sample_tokens: uniform must hold one float32 for '
                         f'each of {n} rows on {dev}, got '
                         f'{tuple(uniform.shape)} {uniform.dtype} on '
                         f'{uniform.device}')
    f32 = torch.float32
    ps = (_param('temperature', temperature, n, dev, f32, 0.0, 1e30),
          _param('top_k', top_k, n, dev, torch.int32, 0, (1 << 31) - 1),
          _param('top_p', top_p, n, dev, f32, 0.0, 1.0),
          _param('min_p', min_p, n, dev, f32, 0.0, 1.0))
    with torch.no_grad():
        if use_hip(logits):
            return hip_required('sample_tokens').sample_tokens(
                logits, uniform.contiguous(), *ps, get_prob)
        return _plain(logits, uniform, *ps, get_prob)


def _plain(logits, uniform, temperature, top_k, top_p, min_p, get_prob):
    n, v = logits.shape

    def col(p):
        t = p if isinstance(p, torch.Tensor) else \
            torch.full((n,), p, dtype=torch.float64, device=logits.device)
        return t.double()[:, None]

    temp, k, p, m = (col(x) for x in (temperature, top_k, top_p, min_p))
    temp, m = temp.clamp(max=1e30), m.clamp(max=1.0)
    if not n:
        return (torch.zeros(0, dtype=torch.int32, device=logits.device),
                torch.zeros(0, device=logits.device) if get_prob else None)
    x = logits.float()
    x = x.masked_fill(torch.isnan(x), -math.inf)
    x, order = torch.sort(x, dim=-1, descending=True, stable=True)
    x, top = x.double(), x[:, :1].double()
    greedy = ~(temp > 0)
    depth = (top - x) / torch.where(greedy, torch.ones_like(temp), temp)
    depth = torch.where(x == top, torch.zeros_like(x), depth)
    w = torch.exp(-depth)
    k = torch.where(greedy, torch.ones_like(k), k)
    at = torch.arange(v, device=x.device)
    w = w.masked_fill((k > 0) & (at >= k), 0.0)
    cum = torch.cumsum(w, -1)
    w = w.masked_fill((p < 1) & (cum - w >= p * cum[:, -1:]) & (at > 0), 0.0)
    w = w.masked_fill((m > 0) & (w < m) & (at > 0), 0.0)
    cum = torch.cumsum(w, -1)
    total = cum[:, -1:]
    u = uniform.double().clamp(0.0, 1.0 - 2.0 ** -24).nan_to_num(
        1.0 - 2.0 ** -24)[:, None]
    pick = (cum <= u * total).sum(-1, keepdim=True).clamp(max=v - 1)
    token = order.gather(1, pick)[:, 0].to(torch.int32)
    none = top[:, 0] == -math.inf
    token = token.masked_fill(none, -1)
    if not get_prob:
        return token, None
    logp = torch.log(w.gather(1, pick) / total)[:, 0].float()
    return token, logp.masked_fill(none, math.nan)
