"""Transformer contrib ops (reference src/operator/contrib/transformer.cc:
650-1038 — interleaved self/enc-dec attention matmuls with fp32-accum
strided-batch GEMM, div_sqrt_dim, sliding-window attention masks).

The batched GEMMs run the native MFMA bgemm; layouts follow the
reference: qkv is [seq, batch, heads*3*head_dim] with per-head
interleaved q,k,v projections.
"""
import math

import torch

from . import nn as _nn
from .dispatch import hip_required, use_hip

__all__ = ['interleaved_matmul_selfatt_qk', 'interleaved_matmul_selfatt_valatt',
           'interleaved_matmul_encdec_qk', 'interleaved_matmul_encdec_valatt',
           'encdec_attention', 'div_sqrt_dim', 'sldwin_atten_mask_like', 'sldwin_atten_score',
           'sldwin_atten_context']


def _split_qkv(qkv, heads):
    # [S, B, H*3*D] -> q,k,v each [B*H, S, D]
    S, B, P = qkv.shape
    D = P // (3 * heads)
    x = qkv.reshape(S, B, heads, 3, D)
    q = x[:, :, :, 0].permute(1, 2, 0, 3).reshape(B * heads, S, D)
    k = x[:, :, :, 1].permute(1, 2, 0, 3).reshape(B * heads, S, D)
    v = x[:, :, :, 2].permute(1, 2, 0, 3).reshape(B * heads, S, D)
    return q.contiguous(), k.contiguous(), v.contiguous(), D


def interleaved_matmul_selfatt_qk(queries_keys_values, heads):
    """[S,B,H*3*D] -> scaled QK^T scores [B*H, S, S]
    (reference transformer.cc:650 _contrib_interleaved_matmul_selfatt_qk)."""
    q, k, _, D = _split_qkv(queries_keys_values, heads)
    scores = _nn.batch_dot(q, k, transpose_b=True)
    return scores / math.sqrt(D)


def interleaved_matmul_selfatt_valatt(queries_keys_values, attention, heads):
    """att [B*H,S,S] x V -> [S, B, H*D] (reference transformer.cc:742)."""
    _, _, v, D = _split_qkv(queries_keys_values, heads)
    S = queries_keys_values.shape[0]
    B = queries_keys_values.shape[1]
    out = _nn.batch_dot(attention.contiguous(), v)          # [B*H, S, D]
    return out.reshape(B, heads, S, D).permute(2, 0, 1, 3) \
              .reshape(S, B, heads * D).contiguous()


def _split_kv(keys_values, heads):
    S, B, P = keys_values.shape
    D = P // (2 * heads)
    x = keys_values.reshape(S, B, heads, 2, D)
    k = x[:, :, :, 0].permute(1, 2, 0, 3).reshape(B * heads, S, D)
    v = x[:, :, :, 1].permute(1, 2, 0, 3).reshape(B * heads, S, D)
    return k.contiguous(), v.contiguous(), D


def interleaved_matmul_encdec_qk(queries, keys_values, heads):
    """queries [Sq,B,H*D], keys_values [Sk,B,H*2*D] -> [B*H,Sq,Sk]."""
    Sq, B, P = queries.shape
    D = P // heads
    q = queries.reshape(Sq, B, heads, D).permute(1, 2, 0, 3) \
               .reshape(B * heads, Sq, D).contiguous()
    k, _, _ = _split_kv(keys_values, heads)
    return _nn.batch_dot(q, k, transpose_b=True) / math.sqrt(D)


def interleaved_matmul_encdec_valatt(keys_values, attention, heads):
    _, v, D = _split_kv(keys_values, heads)
    BH, Sq, _ = attention.shape
    B = keys_values.shape[1]
    out = _nn.batch_dot(attention.contiguous(), v)
    return out.reshape(B, heads, Sq, D).permute(2, 0, 1, 3) \
              .reshape(Sq, B, heads * D).contiguous()


class _EncDecAttention(torch.autograd.Function):
    """The whole attention in one kernel, without stored scores; the
    backward computes them again from each row's log-sum."""

    @staticmethod
    def forward(ctx, q, kv, values, length, mask, heads, kv_heads, tnc):
        ext = hip_required('encdec_attention')
        out, lse = ext.encdec_attention_fwd(
            q, kv, values, heads, kv_heads, length, mask, tnc,
            any(ctx.needs_input_grad[:3]))
        ctx.save_for_backward(q, kv, values, length, mask, out, lse)
        ctx.conf = (heads, kv_heads, tnc)
        return out

    @staticmethod
    @_nn.once_differentiable
    def backward(ctx, dout):
        q, kv, values, length, mask, out, lse = ctx.saved_tensors
        heads, kv_heads, tnc = ctx.conf
        ext = hip_required('encdec_attention')
        dq, dkv, dvalues = ext.encdec_attention_bwd(
            dout, q, kv, values, heads, kv_heads, length, mask, tnc, out, lse)
        return dq, dkv, dvalues, None, None, None, None, None


_ENCDEC_TYPES = (torch.float16, torch.bfloat16, torch.float32)


def _encdec_check(q, kv, values, heads, kv_heads, length, mask, tnc):
    name = 'encdec_attention'
    if q.dtype not in _ENCDEC_TYPES:
        raise TypeError(f'{name}: float16, bfloat16 or float32 queries, got '
                        f'{q.dtype}')
    for t in (kv, values):
        if t is not None and t.dtype != q.dtype:
            raise TypeError(f'{name}: queries of {q.dtype}, keys or values of '
                            f'{t.dtype}')
    for t in (kv, values, length, mask):
        if t is not None and t.device != q.device:
            raise ValueError(f'{name}: queries on {q.device}, another input '
                             f'on {t.device}')
    if q.dim() != 3 or kv.dim() != 3:
        raise ValueError(f'{name}: queries and keys of three axes, got '
                         f'{tuple(q.shape)} and {tuple(kv.shape)}')
    if heads < 1 or kv_heads < 1 or heads % kv_heads:
        raise ValueError(f'{name}: {kv_heads} shared heads do not divide '
                         f'{heads}')
    if q.shape[2] % heads or q.shape[2] < heads:
        raise ValueError(f'{name}: {heads} heads do not divide {q.shape[2]}')
    width = q.shape[2] // heads * kv_heads * (1 if values is not None else 2)
    batch = 1 if tnc else 0
    if kv.shape[2] != width or kv.shape[batch] != q.shape[batch]:
        raise ValueError(f'{name}: queries {tuple(q.shape)} with {heads} '
                         f'heads need keys of {q.shape[batch]} sequences and '
                         f'{width} columns, got {tuple(kv.shape)}')
    if values is not None and values.shape != kv.shape:
        raise ValueError(f'{name}: keys {tuple(kv.shape)} and values '
                         f'{tuple(values.shape)}')
    b, sk = q.shape[batch], kv.shape[1 - batch]
    if length is not None and (length.shape != (b,)
                               or length.dtype not in (torch.int32,
                                                       torch.int64)):
        raise ValueError(f'{name}: valid_length must hold one int32 or int64 '
                         f'for each of {b} sequences, got '
                         f'{tuple(length.shape)} {length.dtype}')
    if mask is not None and (mask.shape != (b, sk)
                             or mask.dtype not in (torch.bool, torch.uint8)):
        raise ValueError(f'{name}: the mask must hold one bool or uint8 for '
                         f'each of {b} x {sk} keys, got {tuple(mask.shape)} '
                         f'{mask.dtype}')
    if q.is_cuda and q.shape[2] // heads > 128:
        raise ValueError(f'{name}: head sizes up to 128 on the GPU, got '
                         f'{q.shape[2] // heads}')


def encdec_attention(queries, keys_values, values=None, heads=1,
                     kv_heads=None, valid_length=None, mask=None,
                     layout='NTC'):
    """softmax(Q K^T / sqrt(D)) V of a decoder's queries over an encoder's
    keys and values, in one kernel (what interleaved_matmul_encdec_qk, a
    masked softmax and interleaved_matmul_encdec_valatt do in three).

    queries [B, Sq, heads*D]; keys_values [B, Sk, kv_heads*2*D], each head's
    key and then its value, or ``keys_values`` the keys and ``values`` the
    values, [B, Sk, kv_heads*D] each.  With ``layout='TNC'`` the first two
    axes are the other way round.  kv_heads (default: heads) divides heads:
    consecutive query heads share one.  Keys from ``valid_length`` [B] on, and
    keys whose ``mask`` [B, Sk] is 0, are left out, whatever their memory
    holds; a row without a key gives zeros.  Returns the queries' shape.
    """
    if layout not in ('NTC', 'TNC'):
        raise ValueError(f'encdec_attention: layout must be NTC or TNC, got '
                         f'{layout!r}')
    heads = int(heads)
    kv_heads = heads if kv_heads is None else int(kv_heads)
    tnc = layout == 'TNC'
    q, kv = queries, keys_values
    _encdec_check(q, kv, values, heads, kv_heads, valid_length, mask, tnc)
    if use_hip(q):
        if valid_length is not None:
            if valid_length.dtype != torch.int32:  # which may not hold all
                valid_length = valid_length.clamp(0, kv.shape[0 if tnc else 1])
            valid_length = valid_length.to(torch.int32).contiguous()
        if mask is not None:
            mask = mask.contiguous()
        q, kv = q.contiguous(), kv.contiguous()
        values = None if values is None else values.contiguous()
        if not _nn.needs_grad(q, kv, values):
            return hip_required('encdec_attention').encdec_attention_fwd(
                q, kv, values, heads, kv_heads, valid_length, mask, tnc,
                False)[0]
        return _EncDecAttention.apply(q, kv, values, valid_length, mask,
                                      heads, kv_heads, tnc)
    if tnc:
        q, kv = q.transpose(0, 1), kv.transpose(0, 1)
        values = None if values is None else values.transpose(0, 1)
    B, sq, sk = q.shape[0], q.shape[1], kv.shape[1]
    D = q.shape[2] // heads
    # [B, kv_heads, rows, D]: the heads that share a key head are its rows
    group = heads // kv_heads
    q = q.float().reshape(B, sq, kv_heads, group, D) \
        .permute(0, 2, 3, 1, 4).reshape(B, kv_heads, group * sq, D)
    if values is None:
        kv = kv.float().reshape(B, sk, kv_heads, 2, D)
        k, v = kv[:, :, :, 0], kv[:, :, :, 1]
    else:
        k, v = (t.float().reshape(B, sk, kv_heads, D) for t in (kv, values))
    keep = torch.ones(B, sk, dtype=torch.bool, device=q.device)
    if valid_length is not None:
        keep = torch.arange(sk, device=q.device) < valid_length[:, None]
    if mask is not None:
        keep = keep & mask.bool()
    k, v = (t.masked_fill(~keep[:, :, None, None], 0.0).permute(0, 2, 1, 3)
            for t in (k, v))
    scores = q @ k.transpose(-1, -2) / math.sqrt(D)
    scores = scores.masked_fill(~keep[:, None, None], float('-inf'))
    some = keep.any(-1)[:, None, None, None]
    # a row without a key: finite scores in place of its own, then zeros
    weights = torch.softmax(scores.masked_fill(~some, 0.0), -1)
    out = (weights.masked_fill(~some, 0.0) @ v) \
        .reshape(B, kv_heads, group, sq, D).permute(0, 3, 1, 2, 4) \
        .reshape(B, sq, heads * D).to(queries.dtype)
    return out.transpose(0, 1).contiguous() if tnc else out


def div_sqrt_dim(data):
    """data / sqrt(last_dim) (reference _contrib_div_sqrt_dim)."""
    return data / math.sqrt(data.shape[-1])


# -- sliding-window (Longformer-style) attention ---------------------------

def sldwin_atten_mask_like(score, dilation, num_heads, w, symmetric=True):
    """Band mask with the same shape as score
    (reference _contrib_sldwin_atten_mask_like transformer.cc:847)."""
    S = score.shape[-2]
    idx = torch.arange(S, device=score.device)
    rel = idx[None, :] - idx[:, None]
    left = w * dilation
    right = w * dilation if symmetric else 0
    band = (rel >= -left) & (rel <= right)
    if dilation > 1:
        band &= (rel % dilation) == 0
    return band.expand_as(score)


def sldwin_atten_score(query, key, dilation, num_heads, w, symmetric=True):
    """Banded QK^T computed densely then masked (the reference stores the
    band compactly; dense+mask is equivalent and MFMA-friendly here)."""
    scores = _nn.batch_dot(query, key, transpose_b=True)
    mask = sldwin_atten_mask_like(scores, dilation, num_heads, w, symmetric)
    return scores.masked_fill(~mask, float('-inf'))


def sldwin_atten_context(score, value, dilation, num_heads, w,
                         symmetric=True):
    return _nn.batch_dot(score.contiguous(), value.contiguous())
