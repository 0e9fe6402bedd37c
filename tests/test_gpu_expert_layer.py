"""The expert layer without rows, and what its roundings are in 16 bits."""
import pytest

pytestmark = pytest.mark.gpu


def test_lookups_in_a_table_without_rows(gpu_handle):
    """for no token there is nothing to look up, and nothing to add to a gradient; with tokens such a table is refused"""
    import torch
    import mluop_hip
    none = torch.zeros(0, dtype=torch.int32, device="cuda")
    for dtype in (torch.float32, torch.bfloat16):
        table = torch.zeros(0, 24, dtype=dtype, device="cuda")
        out = mluop_hip.embedding_forward(gpu_handle, table, none.view(0, 2))
        assert out.shape == (0, 2, 24) and out.dtype == dtype
        grad = mluop_hip.embedding_backward(gpu_handle, out, none.view(0, 2), 0)
        assert grad.shape == (0, 24) and grad.dtype == dtype
        with pytest.raises(mluop_hip.MluOpError):
            mluop_hip.embedding_forward(gpu_handle, table, torch.zeros(1, dtype=torch.int32, device="cuda"))


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_no_rows(dtype):
    import torch
    from mluop_hip import nn as spnn
    dtype = getattr(torch, dtype)
    layer = spnn.ExpertMLP(24, 40, experts=5, choices=2).cuda()
    x = torch.zeros(0, 24, device="cuda", dtype=dtype, requires_grad=True)
    out = layer(x)
    assert out.shape == (0, 24) and out.dtype == dtype
    grads = torch.autograd.grad(out, [x] + list(layer.parameters()), torch.zeros_like(out))
    assert grads[0].shape == (0, 24)
    for g, p in zip(grads[1:], layer.parameters()):
        assert g.shape == p.shape and not bool(g.any())


def test_order_of_no_rows():
    import torch
    from mluop_hip import nn as spnn
    for shape in ((0, 2), (0,), (0, 0), (3, 0)):
        chosen = torch.zeros(shape, dtype=torch.int64, device="cuda")
        rows, starts, places = spnn.expert_order(chosen, 4)
        assert rows.shape == (0,) and rows.dtype == torch.int32 and starts.tolist() == [0] * 5
        assert places.shape[0] == shape[0] and places.numel() == 0
    rows, starts, places = spnn.expert_order(torch.tensor([2, 0, 2], device="cuda"), 3)
    assert rows.tolist() == [1, 0, 2] and starts.tolist() == [0, 1, 1, 3] and places.tolist() == [[1], [0], [2]]


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("choices", [1, 2, 6])
def test_results_are_weighed_and_added_in_32_bits(dtype, choices):
    """the second layer's rows are given, so that what is left is sum of weight * row and one rounding"""
    import torch
    from mluop_hip import nn as spnn
    dtype = getattr(torch, dtype)
    torch.manual_seed(choices)
    layer = spnn.ExpertMLP(32, 16, experts=8, choices=choices).cuda()
    x = torch.randn(500, 32, device="cuda").to(dtype)
    rows = {}
    layer.down.register_forward_hook(lambda module, args, out: rows.setdefault("out", out))
    out = layer(x)
    assert out.dtype == dtype
    scores, chosen = torch.topk(layer.gate(x.float()), choices, dim=1)
    places = spnn.expert_order(chosen, 8)[2].long()
    terms = rows["out"].double()[places] * torch.softmax(scores.double(), dim=1).unsqueeze(2)
    want, size = terms.sum(dim=1), terms.abs().sum(dim=1)
    last = 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -11
    # scores and softmax in fp32 (a score of a few units: its exponential is off by some units in the last place), products
    # and sums
    room = (choices + 32) * 2.0 ** -23 * size + last * want.abs() + 2.0 ** -25
    assert bool(((out.double() - want).abs() <= room).all())
