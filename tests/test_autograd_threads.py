"""Which thread runs a backward pass, and that its gradients do not change."""
import threading

import pytest
import torch

import mxnet_amd as mx
from mxnet_amd import autograd


class _Note(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, seen):
        ctx.seen = seen
        return x * 2

    @staticmethod
    def backward(ctx, dy):
        ctx.seen.append(threading.get_ident())
        return dy * 2, None


@pytest.mark.parametrize('device', [
    'cpu', pytest.param('cuda:0', marks=pytest.mark.gpu)])
def test_one_device_runs_in_the_calling_thread(device):
    seen = []
    x = torch.ones(4, device=device, requires_grad=True)
    before = torch._C._is_multithreading_enabled()
    with autograd.record():
        y = mx.nd.from_torch(_Note.apply(x, seen))
    y.backward()
    with autograd.record():
        y = mx.nd.from_torch(_Note.apply(x, seen))
    g = autograd.grad([y], [mx.nd.from_torch(x)])[0]
    assert seen == [threading.get_ident()] * 2
    assert torch.equal(x.grad, torch.full_like(x, 2))
    assert torch.equal(g.to_torch(), torch.full_like(x, 2))
    assert torch._C._is_multithreading_enabled() == before


@pytest.mark.gpu
def test_heads_on_two_devices():
    """Heads on a CPU and a GPU in one pass, and a pass within a pass."""
    a = torch.ones(3, requires_grad=True)
    b = torch.ones(3, device='cuda:0', requires_grad=True)
    with autograd.record():
        heads = [mx.nd.from_torch(a * 3), mx.nd.from_torch(b * 4)]
    autograd.backward(heads)
    assert torch.equal(a.grad, torch.full_like(a, 3))
    assert torch.equal(b.grad, torch.full_like(b, 4))

    class Inner(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x):
            ctx.save_for_backward(x)
            return x * x

        @staticmethod
        def backward(ctx, dy):
            x, = ctx.saved_tensors
            with torch.enable_grad():
                z = x.detach().requires_grad_()
                y = mx.nd.from_torch(z * z)
            y.backward()
            return dy * z.grad

    c = torch.full((3,), 5.0, device='cuda:0', requires_grad=True)
    with autograd.record():
        y = mx.nd.from_torch(Inner.apply(c))
    y.backward()
    assert torch.equal(c.grad, torch.full_like(c, 10))


class _Head:
    is_cuda = True

    def __init__(self, index):
        self.device = torch.device('cuda', index)

    def get_device(self):
        return self.device.index


@pytest.mark.parametrize('used,heads,alone', [
    ({0}, [0], True), ({0}, [0, 0], True), ({1}, [1], True),
    ({0, 1}, [0], False), ({0, 2}, [2], False), ({0, 1}, [0, 1], False)])
def test_a_process_of_several_gpus_keeps_its_threads(monkeypatch, used, heads,
                                                     alone):
    """Layers may lie on any GPU that the process has worked on, wherever
    the heads are."""
    monkeypatch.setattr(torch.cuda, 'device_count', lambda: 3)
    monkeypatch.setattr(torch._C, '_cuda_hasPrimaryContext',
                        lambda i: i in used)
    before = torch._C._is_multithreading_enabled()
    with autograd._engine_threads([_Head(i) for i in heads]):
        assert torch._C._is_multithreading_enabled() == (before and not alone)
    assert torch._C._is_multithreading_enabled() == before


def test_the_state_comes_back_after_an_error(monkeypatch):
    monkeypatch.setattr(torch.cuda, 'device_count', lambda: 1)
    before = torch._C._is_multithreading_enabled()
    with autograd.record():
        with pytest.raises(ZeroDivisionError):
            with autograd._engine_threads([_Head(0)]):
                assert not autograd.is_recording()
                assert not autograd.is_training()
                1 / 0
        assert autograd.is_recording() and autograd.is_training()
    assert not autograd.is_recording()
    assert torch._C._is_multithreading_enabled() == before


class _State(mx.operator.CustomOp):
    seen = []

    def forward(self, is_train, req, in_data, out_data, aux):
        self.assign(out_data[0], req[0], in_data[0] * 2)

    def backward(self, req, out_grad, in_data, out_data, in_grad, aux):
        self.seen.append((autograd.is_recording(), autograd.is_training()))
        self.assign(in_grad[0], req[0], out_grad[0] * 2)


@mx.operator.register('state_of_the_backward_pass')
class _StateProp(mx.operator.CustomOpProp):
    def create_operator(self, ctx, shapes, dtypes):
        return _State()


@pytest.mark.gpu
def test_custom_backward_neither_records_nor_trains():
    """As in a thread of the device, also where the caller records."""
    x = torch.ones(4, device='cuda:0', requires_grad=True)
    a = mx.nd.from_torch(x)
    _State.seen.clear()
    with autograd.record():
        mx.nd.Custom(a, op_type='state_of_the_backward_pass').backward()
        y = mx.nd.Custom(a, op_type='state_of_the_backward_pass')
        autograd.grad([y], [a])
        assert autograd.is_recording() and autograd.is_training()
    mx.nd.Custom(a, op_type='state_of_the_backward_pass').backward()
    assert _State.seen == [(False, False)] * 3
    assert torch.equal(x.grad, torch.full_like(x, 4))
