"""Group norm on the paths of many rows: starts that make no sense on both sides of the line between moments joined by the
pass that applies them and by their own launch, and results that go past the caches."""
import pytest

from launches import launched

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,channels,joined", [(5000, 16, False), (9000, 8, False), (60_000, 64, True), (30_000, 20, None)])
def test_starts_that_make_no_sense_stay_in_bounds(gpu_handle, rows, channels, joined):
    """(their results are undefined; no access leaves a tensor: outputs and workspaces lie between guard bands)"""
    import torch
    import mluop_hip
    print("starts", rows, channels, flush=True)
    g = torch.Generator(device="cuda").manual_seed(rows)
    x = torch.randn(rows, channels, device="cuda", generator=g).half()
    dy = torch.randn(rows, channels, device="cuda", generator=g).half()
    w = torch.ones(channels, device="cuda")
    for starts in ([0, rows, 0, rows, 0, rows], [-7, 1 << 30, 5, 4, 3, 2], [9] * 6, [rows, 0, -1, rows, 0, 1],
                   [0] + [rows, 0] * 30 + [rows], [(1 << 31) - 1, -(1 << 31)] * 4):
        dev = torch.tensor(starts, dtype=torch.int32, device="cuda")
        (_, mean, rstd), names = launched(gpu_handle, lambda: mluop_hip.group_norm_forward(gpu_handle, x, w, w, 4, dev))
        assert names[0] == "groupNormMoments"
        if joined is not None:
            assert ("groupNormJoinMoments" in names) == joined
        _, names = launched(gpu_handle, lambda: mluop_hip.group_norm_backward(gpu_handle, dy, x, w, w, mean, rstd, 4, dev))
        assert names[0] == "groupNormGradSums"
    torch.cuda.synchronize()


# (groups narrower than a vector, as wide, and wider)
@pytest.mark.parametrize("dtype,channels,groups", [("float16", 48, 16), ("bfloat16", 32, 8), ("float32", 24, 2),
                                                   ("float16", 33, 3)])
def test_results_past_the_caches(gpu_handle, dtype, channels, groups):
    """32 MB of results or more, samples of several tiles, of one row and of none, rows of no sample"""
    import torch
    import mluop_hip
    dtype = getattr(torch, dtype)
    rows = (33 << 20) // (channels * dtype.itemsize) + 1001
    starts = [13, 13, 14, rows // 3, rows // 3 + 700, rows - 5]
    dev = torch.tensor(starts, dtype=torch.int32, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(channels)
    x = (torch.randn(rows, channels, device="cuda", generator=g) + torch.randn(channels, device="cuda", generator=g)).to(dtype)
    dy = torch.randn(rows, channels, device="cuda", generator=g).to(dtype)
    w = 1 + 0.3 * torch.randn(channels, device="cuda", generator=g)
    b = 0.3 * torch.randn(channels, device="cuda", generator=g)
    out, mean, rstd = mluop_hip.group_norm_forward(gpu_handle, x, w, b, groups, dev, 1e-5, "silu")
    dx, dw, db = mluop_hip.group_norm_backward(gpu_handle, dy, x, w, b, mean, rstd, groups, dev, "silu")
    last = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}[dtype]
    want_dw, want_db = (torch.zeros(channels, dtype=torch.float64, device="cuda") for _ in range(2))
    # sums of n values of size s in fp32, in trees over runs of up to a thousand: 2^-18 of s a mean; values of up to some 8
    for s, (lo, hi) in enumerate(zip(starts, starts[1:])):
        if lo == hi:
            continue
        v = x[lo:hi].double().view(hi - lo, groups, -1)
        m = v.mean(dim=(0, 2))
        r = (v.var(dim=(0, 2), unbiased=False) + 1e-5) ** -0.5
        spread = float(r.max())
        assert float((mean[s].double() - m).abs().max()) <= 2.0 ** -18 * 8
        assert float((rstd[s].double() / r - 1).abs().max()) <= 2.0 ** -14
        normed = ((v - m[:, None]) * r[:, None]).view(hi - lo, channels)
        z = normed * w.double() + b.double()
        t = torch.sigmoid(z)
        z_room = 2.0 ** -14 * (1 + normed.abs() * w.double().abs()) + 2.0 ** -17 * spread
        y = z * t
        assert bool(((out[lo:hi].double() - y).abs() <= last * y.abs() + 1.2 * z_room + 2.0 ** -24).all())
        dz = dy[lo:hi].double() * (t * (1 + z * (1 - t)))
        want_dw += (dz * normed).sum(dim=0)
        want_db += dz.sum(dim=0)
        d = (dz * w.double()).view(hi - lo, groups, -1)
        n = normed.view(hi - lo, groups, -1)
        d = d - d.mean(dim=(0, 2), keepdim=True) - n * (d * n).mean(dim=(0, 2), keepdim=True)
        d = (d * r[:, None]).view(hi - lo, channels)
        room = 2.0 ** -12 * spread * (dy[lo:hi].double().abs() + 1) * (1 + normed.abs())
        assert bool(((dx[lo:hi].double() - d).abs() <= last * d.abs() + room + 2.0 ** -24).all())
    for t in (out, dx):
        assert not bool(t[:starts[0]].any()) and not bool(t[starts[-1]:].any())
    for got, want in ((dw, want_dw), (db, want_db)):
        assert bool(((got.double() - want).abs() <= 2.0 ** -14 * (rows ** 0.5 * 8 + want.abs())).all())
