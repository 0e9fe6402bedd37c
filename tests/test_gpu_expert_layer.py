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
