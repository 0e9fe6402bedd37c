"""The layers of a residual block take a SparseTensor or rows: the same results, and the tensor's coordinates."""
import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("which", ["norm", "scan", "experts", "dropout"])
def test_a_sparse_tensor_or_its_rows(which):
    import torch
    from mluop_hip import nn as spnn
    torch.manual_seed(0)
    make = {"norm": lambda: spnn.LayerNorm(32), "scan": lambda: spnn.GatedScan(32), "experts": lambda: spnn.ExpertMLP(32, 48, 5, 2),
            "dropout": lambda: spnn.DropoutAdd(0.3)}
    layer = make[which]().cuda()
    sizes = (7, 12)
    indices = torch.tensor([[n, 0, 0, i] for n, size in enumerate(sizes) for i in range(size)], dtype=torch.int32, device="cuda")
    rows = torch.randn(sum(sizes), 32, device="cuda")
    before = {k: v.clone() for k, v in layer.state_dict().items()}
    got = layer(spnn.SparseTensor(rows, indices, (1, 1, 16), 2, distinct=True, ordered=True))
    layer.load_state_dict(before)
    starts = torch.tensor([0, 7, 19], dtype=torch.int32, device="cuda")
    want = layer(rows, starts) if which == "scan" else layer(rows)
    assert isinstance(got, spnn.SparseTensor) and torch.equal(got.indices, indices)
    assert torch.equal(got.features, want)
