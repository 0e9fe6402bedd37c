"""Layers whose weights lie on another device than their features refuse the call."""
import pytest

pytestmark = pytest.mark.gpu


def test_weights_that_were_left_on_the_host():
    import torch
    from mluop_hip import nn as spnn
    idx = torch.tensor([[0, 0, i // 5, i % 5] for i in range(15)], dtype=torch.int32, device="cuda")
    x = spnn.SparseTensor(torch.randn(15, 32, device="cuda"), idx, (1, 5, 5), 1, distinct=True)
    for layer in (spnn.SubMConv3d(32, 32, 3), spnn.GroupNormAct(4, 32), spnn.LayerNorm(32)):
        with pytest.raises(ValueError):
            layer(x)
        assert layer.cuda()(x).features.shape == (15, 32)
