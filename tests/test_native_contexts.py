"""An operator of the native runtime takes arrays of one device."""
import numpy as np
import pytest

import mxnet_amd as mx
from mxnet_amd import _core, autograd
from mxnet_amd.base import set_native


@pytest.fixture
def native():
    prev = set_native(True)
    yield
    set_native(prev)


def cpu(*shape, dtype='float32'):
    return mx.nd.array(np.ones(shape), dtype=dtype)


def far(*shape, dtype='float32', index=0):
    """An array of a GPU that has no memory yet, so that none is needed."""
    flag = {'float32': 0, 'int32': 4, 'int64': 6, 'uint8': 3}[dtype]
    return mx.nd.NDArray(_core.NDArray(list(shape), 2, index, flag,
                                     delay_alloc=True))


def calls(a, b):
    """Calls with one array by `b`, the others by `a`."""
    att = mx.nd.contrib.encdec_attention
    draw = mx.nd.contrib.sample_tokens
    norm = mx.nd.RMSNorm
    return [
        lambda: norm(a(2, 8), b(8)),
        lambda: norm(a(2, 8), a(8), residual=b(2, 8)),
        lambda: norm(b(2, 8), a(8), out_type='int8'),
        lambda: att(a(1, 2, 8), b(1, 3, 16)),
        lambda: att(a(1, 2, 8), a(1, 3, 8), b(1, 3, 8)),
        lambda: att(a(1, 2, 8), a(1, 3, 16), valid_length=b(1, dtype='int64')),
        lambda: att(a(1, 2, 8), a(1, 3, 16), mask=b(1, 3, dtype='uint8')),
        lambda: draw(a(2, 8), b(2)),
        lambda: draw(a(2, 8), a(2), temperature=b(2)),
        lambda: draw(a(2, 8), a(2), top_k=b(2, dtype='int32')),
        lambda: a(2, 8) + b(2, 8),
    ]


@pytest.mark.parametrize('i', range(11))
def test_arrays_of_two_devices_are_refused(native, i):
    others = [(far, cpu), (cpu, far),
              (far, lambda *s, **kw: far(*s, index=1, **kw))]
    for a, b in others:
        with pytest.raises(RuntimeError, match='is given an array on'):
            calls(a, b)[i]()
        with autograd.record():
            with pytest.raises(RuntimeError, match='is given an array on'):
                calls(a, b)[i]()
    calls(cpu, cpu)[i]()


@pytest.mark.gpu
def test_on_the_gpu(native):
    x = mx.nd.array(np.ones((2, 8)), ctx=mx.gpu(0), dtype='float32')
    with pytest.raises(RuntimeError, match='is given an array on'):
        mx.nd.RMSNorm(x, cpu(8))
    y = mx.nd.RMSNorm(x, cpu(8).as_in_context(mx.gpu(0)))
    assert np.allclose(y.asnumpy(), 1, atol=1e-5)
