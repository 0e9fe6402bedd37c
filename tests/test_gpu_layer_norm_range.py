"""Layer norm of rows whose squared differences leave fp32's range: rstd is zero and the result the bias; rows beside them are as
ever."""
import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("channels", [8, 33, 1024])
def test_rows_far_apart(gpu_handle, dtype, channels):
    import torch
    import mluop_hip
    g = torch.Generator(device="cuda").manual_seed(channels)
    x = torch.randn(5, channels, device="cuda", generator=g).to(getattr(torch, dtype))
    # (sums stay finite, squares of 2^100 do not)
    wide = torch.where(torch.arange(channels, device="cuda") % 2 == 0, 1.0, -1.0) * 2.0 ** 100
    far = x.clone()
    far[2] = wide.to(x.dtype)
    w, b = 1 + torch.rand(channels, device="cuda", generator=g), torch.randn(channels, device="cuda", generator=g)
    out, mean, rstd = mluop_hip.layer_norm_forward(gpu_handle, far, w, b)
    ref, _, ref_rstd = mluop_hip.layer_norm_forward(gpu_handle, x, w, b)
    others = torch.tensor([0, 1, 3, 4], device="cuda")
    assert float(rstd[2]) == 0.0 and torch.equal(out[2], b.to(x.dtype))
    assert torch.equal(out[others], ref[others]) and torch.equal(rstd[others], ref_rstd[others])
    dx, dw, db = mluop_hip.layer_norm_backward(gpu_handle, torch.ones_like(far), far, w, b, mean, rstd)
    assert not bool(dx[2].any()) and bool(dw.isfinite().all()) and bool((db == 5).all())
