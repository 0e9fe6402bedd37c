"""The group norm's layer without a weight, a bias or both: values and gradients."""
import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("weight,bias", [(False, False), (True, False), (False, True)])
def test_group_norm_without_weight_or_bias(weight, bias):
    import torch
    from mluop_hip import nn as spnn
    g = torch.Generator(device="cuda").manual_seed(0)

    def randn(*shape):
        return torch.randn(*shape, device="cuda", generator=g).requires_grad_()
    x, w, b = randn(90, 24), randn(24) if weight else None, randn(24) if bias else None
    leaves = [t for t in (x, w, b) if t is not None]
    got = spnn.group_norm(x, w, b, 4)
    # (torch's own gradient wants both)
    want = torch.nn.functional.group_norm(x.t()[None], 4, torch.ones(24, device="cuda") if w is None else w,
                                          torch.zeros(24, device="cuda") if b is None else b, 1e-5)[0].t()
    assert torch.allclose(got, want, atol=1e-5)
    dy = torch.randn(90, 24, device="cuda", generator=g)
    for a, c in zip(torch.autograd.grad(got, leaves, dy), torch.autograd.grad(want, leaves, dy)):
        assert torch.allclose(a, c, rtol=1e-4, atol=1e-4)


def test_layer_without_params():
    import torch
    from mluop_hip import nn as spnn
    layer = spnn.GroupNormAct(4, 24, affine=False, activation="relu").cuda()
    x = torch.randn(50, 24, device="cuda", requires_grad=True)
    layer(x).sum().backward()
    assert not list(layer.parameters()) and bool(torch.isfinite(x.grad).all())
