"""mx.sym.contrib: nd.contrib's operators as graph nodes, so that
``F.contrib`` is the same in both modes of ``hybrid_forward``."""

__all__ = ['encdec_attention', 'sample_tokens']


def _node(op, inputs, name, attrs):
    from . import _make_op
    return _make_op(op)(*inputs, name=name, **{
        k: v for k, v in attrs.items() if v is not None})


def encdec_attention(queries, keys_values, values=None, heads=1,
                     kv_heads=None, valid_length=None, mask=None,
                     layout='NTC', name=None):
    """nd.contrib.encdec_attention as a graph node."""
    return _node('_contrib_encdec_attention', [queries, keys_values], name,
                 dict(values=values, heads=heads, kv_heads=kv_heads,
                      valid_length=valid_length, mask=mask, layout=layout))


def sample_tokens(logits, uniform, temperature=1.0, top_k=0, top_p=1.0,
                  min_p=0.0, get_prob=False, name=None):
    """nd.contrib.sample_tokens as a graph node (with ``get_prob`` a list of
    two Symbols); parameters are numbers or Symbols."""
    from . import Symbol
    out = _node('_contrib_sample_tokens', [logits, uniform], name,
                dict(temperature=temperature, top_k=top_k, top_p=top_p,
                     min_p=min_p, get_prob=get_prob))
    if not get_prob:
        return out
    out._node.num_outputs = 2
    return [Symbol(out._node, i) for i in range(2)]


def _evaluate(name):
    """What a node of that operator runs: nd.contrib is imported at the call,
    since it needs this package."""
    def run(*args, **kwargs):
        from ..ndarray import contrib
        return getattr(contrib, name)(*args, **kwargs)
    return run


EVAL = {'_contrib_' + n: _evaluate(n) for n in __all__}
