"""A module that counts its calls, run again inside of a backward pass: refused where it drops, as it is where it does not; the
function with a state of the caller's drops the same elements both times."""
import pytest


def run_again(layer):
    """an identity whose backward pass calls the layer, as a checkpoint's does"""
    import torch

    class Again(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x):
            return x.clone()

        @staticmethod
        def backward(ctx, dy):
            return layer(dy)
    return Again.apply


def test_refused_before_anything_is_counted():
    import torch
    from mluop_hip import nn as spnn
    layer = spnn.DropoutAdd(0.5, seed=3)
    x = torch.randn(4, 5, requires_grad=True)
    with pytest.raises(RuntimeError, match="backward pass would drop other elements"):
        run_again(layer)(x).sum().backward()
    assert layer.state.tolist() == [3, 0]


@pytest.mark.parametrize("p,training", [(0.0, True), (0.5, False)])
def test_what_drops_nothing_is_not_refused(p, training):
    import torch
    from mluop_hip import nn as spnn
    layer = spnn.DropoutAdd(p).train(training)
    x = torch.randn(4, 5, requires_grad=True)
    run_again(layer)(x).sum().backward()
    assert torch.equal(x.grad, torch.ones_like(x))


@pytest.mark.gpu
@pytest.mark.parametrize("reentrant", [False, True])
def test_checkpoints(reentrant):
    import torch
    from torch.utils.checkpoint import checkpoint
    from mluop_hip import nn as spnn
    layer = spnn.DropoutAdd(0.5, seed=1).cuda()
    x = torch.randn(2000, 16, device="cuda", requires_grad=True)
    with pytest.raises(RuntimeError, match="backward pass would drop other elements"):
        checkpoint(lambda t: layer(t.tanh()), x, use_reentrant=reentrant).sum().backward()
    state = torch.tensor([1, 7], device="cuda")

    def f(t):
        return spnn.dropout_add(t.tanh(), t, 0.5, state).square().sum()
    (want,) = torch.autograd.grad(f(x), x)
    x.grad = None
    checkpoint(f, x, use_reentrant=reentrant).backward()
    assert torch.equal(x.grad, want)
