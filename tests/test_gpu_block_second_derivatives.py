"""The nodes of a residual block's operators are differentiable once: a derivative of their gradients is refused, never left out of
a sum."""
import pytest

pytestmark = pytest.mark.gpu


def operators():
    """{name: (function of one tensor, that tensor)}"""
    import torch
    from mluop_hip import nn as spnn
    g = torch.Generator(device="cuda").manual_seed(0)

    def randn(*shape):
        return torch.randn(*shape, device="cuda", generator=g)
    x, gates, initial = randn(20, 8), randn(20, 8), randn(3, 8)
    starts = torch.tensor([0, 7, 7, 20], dtype=torch.int32, device="cuda")
    weight, bias = randn(8), randn(8)
    _, first, places = spnn.expert_order(torch.arange(40, device="cuda").view(20, 2) % 3, 3)
    weights, results = randn(20, 2), randn(40, 8)
    state = torch.tensor([5, 6], device="cuda")
    return {"norm": (lambda t: spnn.layer_norm(t, weight, bias), x),
            "norm's weight": (lambda t: spnn.layer_norm(x, t, None), weight),
            "recurrence": (lambda t: spnn.gated_scan(t, gates, starts, initial)[0], x),
            "recurrence's gates": (lambda t: spnn.gated_scan(x, t, starts, initial, "exp", True)[0], -gates.abs()),
            "recurrence's states": (lambda t: spnn.gated_scan(x, gates, starts, t)[1], initial),
            "dispatch": (lambda t: spnn.expert_dispatch(t, places, first), x),
            "combine": (lambda t: spnn.expert_combine(t, places, first, weights), results),
            "combine's weights": (lambda t: spnn.expert_combine(results, places, first, t), weights),
            "dropout": (lambda t: spnn.dropout_add(t, x, 0.25, state), x),
            "dropout's residual": (lambda t: spnn.dropout_add(x, t, 0.25, state), x)}


NAMES = ["norm", "norm's weight", "recurrence", "recurrence's gates", "recurrence's states", "dispatch", "combine",
         "combine's weights", "dropout", "dropout's residual"]


@pytest.mark.parametrize("name", NAMES)
def test_a_second_derivative_is_refused(name):
    import torch
    f, t = operators()[name]
    t = t.clone().requires_grad_()
    (plain,) = torch.autograd.grad(f(t).square().sum(), t)
    (first,) = torch.autograd.grad(f(t).square().sum(), t, create_graph=True)
    assert torch.equal(plain, first)
    with pytest.raises(RuntimeError, match="twice"):
        (first.square().sum() + t.sum()).backward()


@pytest.mark.parametrize("name", ["norm", "recurrence's gates"])
def test_where_only_the_inputs_bring_a_derivative(name):
    """a gradient of ones has none itself, but the slope depends on the inputs"""
    import torch
    f, t = operators()[name]
    t = t.clone().requires_grad_()
    (first,) = torch.autograd.grad(f(t).sum(), t, create_graph=True)
    with pytest.raises(RuntimeError, match="twice"):
        (first.square().sum() + t.sum()).backward()


@pytest.mark.parametrize("name", ["dispatch", "dropout", "dropout's residual"])
def test_what_has_no_second_derivative_is_not_refused(name):
    import torch
    f, t = operators()[name]
    t = t.clone().requires_grad_()
    (first,) = torch.autograd.grad(f(t).sum(), t, create_graph=True)
    (first.sum() + t.square().sum()).backward()
    assert torch.equal(t.grad, 2 * t.detach())
