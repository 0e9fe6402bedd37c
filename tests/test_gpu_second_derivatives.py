"""The library's nodes are differentiable once: a derivative of their gradients is refused, never left out of a sum."""
import pytest

pytestmark = pytest.mark.gpu


def operators():
    """(name, function of one tensor, that tensor)"""
    import torch
    from mluop_hip import nn as spnn
    g = torch.Generator(device="cuda").manual_seed(0)

    def randn(*shape):
        return torch.randn(*shape, device="cuda", generator=g)
    tokens = torch.randint(0, 9, (30,), device="cuda", generator=g)
    starts = torch.tensor([0, 7, 20], dtype=torch.int32, device="cuda")
    x, w = randn(20, 8), randn(2, 8, 6)
    weight, bias = randn(8), randn(8)
    cells = torch.tensor([[0, 0, i // 5, i % 5] for i in range(20)], dtype=torch.int32, device="cuda")
    conv = spnn.SubMConv3d(8, 4, 3).cuda()
    return [("embedding", lambda t: spnn.embedding(t, tokens, 0.5), randn(9, 5)),
            ("rows", lambda t: spnn.grouped_matmul(t, w.clone().requires_grad_(), starts), x),
            ("filters", lambda t: spnn.grouped_matmul(x, t, starts), w),
            ("norm", lambda t: spnn.group_norm(t, weight, bias, 2, starts, activation="silu"), x),
            ("norm's weight", lambda t: spnn.group_norm(x, t, bias, 2, starts, activation="silu"), weight),
            ("convolution", lambda t: conv(spnn.SparseTensor(t, cells, (1, 5, 5), 1, distinct=True)).features, x)]


@pytest.mark.parametrize("which", range(6))
def test_a_second_derivative_is_refused(which):
    import torch
    name, f, t = operators()[which]
    print(name, flush=True)
    t = t.clone().requires_grad_()
    (plain,) = torch.autograd.grad(f(t).square().sum(), t)
    (first,) = torch.autograd.grad(f(t).square().sum(), t, create_graph=True)
    assert torch.equal(plain, first)
    with pytest.raises(RuntimeError, match="twice"):
        (first.square().sum() + t.sum()).backward()


def test_where_only_the_inputs_bring_a_derivative():
    """a gradient of ones has none itself, but the norm's slope depends on the features"""
    import torch
    name, f, t = operators()[3]
    t = t.clone().requires_grad_()
    (first,) = torch.autograd.grad(f(t).sum(), t, create_graph=True)
    with pytest.raises(RuntimeError, match="twice"):
        (first.square().sum() + t.sum()).backward()


def test_what_has_no_second_derivative_is_not_refused():
    """the lookup is linear: a gradient of ones gives a constant"""
    import torch
    name, f, t = operators()[0]
    t = t.clone().requires_grad_()
    (first,) = torch.autograd.grad(f(t).sum(), t, create_graph=True)
    (first.sum() + t.square().sum()).backward()
    assert torch.equal(t.grad, 2 * t.detach())
