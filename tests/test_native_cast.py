"""The native runtime's cast, against numpy's."""
import numpy as np
import pytest

import mxnet_amd as mx
from mxnet_amd.base import set_native

DEVICES = ['cpu', pytest.param('gpu', marks=pytest.mark.gpu)]
WHOLE = {'int8': (-128, 127), 'uint8': (0, 255),
         'int32': (-(1 << 31), (1 << 31) - 1),
         'int64': (-(1 << 63), (1 << 63) - 1)}


@pytest.fixture
def native():
    prev = set_native(True)
    yield
    set_native(prev)


def cast(a, dtype, device):
    x = mx.nd.array(a, ctx=mx.cpu() if device == 'cpu' else mx.gpu(0),
                    dtype=str(a.dtype))
    assert x.is_native
    return x.astype(dtype).asnumpy()


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('to', list(WHOLE))
@pytest.mark.parametrize('of', list(WHOLE))
def test_whole_numbers(native, of, to, device):
    """What both types hold comes through as it is, and what the second does
    not hold loses its upper bits."""
    lo, hi = WHOLE[of]
    values = [0, 1, 100, 127, -1, -128, 255, (1 << 24) + 1, -(1 << 24) - 3,
              (1 << 31) - 1, -(1 << 31), (1 << 40) + 5, lo, hi, hi - 1]
    a = np.array([v for v in values if lo <= v <= hi], of)
    got = cast(a, to, device)
    assert str(got.dtype) == to and np.array_equal(got, a.astype(to))


@pytest.mark.parametrize('device', DEVICES)
def test_float64(native, device):
    a = np.array([0.1, -3.7, 1e300, 2.0 ** 40 + 0.25, 7.0])
    assert np.array_equal(cast(a[[0, 1, 3, 4]], 'float32', device),
                          a[[0, 1, 3, 4]].astype('float32'))
    assert np.array_equal(cast(a, 'float64', device), a)
    assert np.array_equal(cast(a[[1, 3, 4]], 'int64', device),
                          a[[1, 3, 4]].astype('int64'))
    whole = np.array([(1 << 53) - 1, -(1 << 30) - 1], 'int64')
    assert np.array_equal(cast(whole, 'float64', device),
                          whole.astype('float64'))


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('of', list(WHOLE) + ['float16', 'float32', 'float64'])
def test_small_values_in_every_type(native, of, device):
    a = np.arange(0, 60, 3).astype(of)
    for to in list(WHOLE) + ['float16', 'float32', 'float64']:
        assert np.array_equal(cast(a, to, device), a.astype(to))
