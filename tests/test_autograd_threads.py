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
