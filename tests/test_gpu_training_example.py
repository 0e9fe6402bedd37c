"""The operators of a training step together: the example learns, its expert layer is the formula's, and one row goes the
way of a batch."""
import importlib.util
import os

import pytest

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def example():
    spec = importlib.util.spec_from_file_location("voxel_experts", os.path.join(ROOT, "examples", "voxel_experts.py"))
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def test_the_example_learns():
    import torch
    _, losses = example().train(40, 6000, torch.bfloat16)
    assert sum(losses[-4:]) / 4 < 0.7 * sum(losses[:4]) / 4


@pytest.mark.parametrize("rows", [1, 7, 300])
def test_expert_layer(rows):
    import torch
    from mluop_hip import nn as spnn
    torch.manual_seed(rows)
    layer = spnn.ExpertMLP(24, 40, experts=5, choices=2).cuda()
    x = torch.randn(rows, 24, device="cuda", requires_grad=True)
    out = layer(x)
    scores = x @ layer.gate.weight.t()
    top, chosen = torch.topk(scores, 2, dim=1)
    weight = torch.zeros_like(scores).scatter(1, chosen, torch.softmax(top, dim=1))
    ref = sum(weight[:, e:e + 1] * (torch.nn.functional.silu(x @ layer.up.weight[e]) @ layer.down.weight[e])
              for e in range(5))
    assert torch.allclose(out, ref, atol=1e-5)
    dy = torch.randn_like(out)
    inputs = [x] + list(layer.parameters())
    for a, b in zip(torch.autograd.grad(out, inputs, dy), torch.autograd.grad(ref, inputs, dy)):
        assert torch.allclose(a, b, atol=1e-4 * (1 + float(b.abs().max())))


def test_expert_order():
    import torch
    from mluop_hip import nn as spnn
    chosen = torch.tensor([[2, 0], [0, 1], [2, 3]], device="cuda")
    rows, starts, places = spnn.expert_order(chosen, 5)
    assert rows.tolist() == [0, 1, 1, 0, 2, 2] and starts.tolist() == [0, 2, 3, 5, 6, 6]
    assert places.tolist() == [[3, 0], [1, 2], [4, 5]]
