"""Rows of few channels through the operators of a residual block: threads that share a row are fewer, and rows share lines."""
import pytest

from test_gpu_expert_rows import LAST, LEAST, routing, taken

pytestmark = pytest.mark.gpu

CHANNELS = [1, 2, 4, 7, 8, 12, 16, 24, 31, 32, 33, 48]


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("channels", CHANNELS)
def test_norm(gpu_handle, dtype, channels):
    import torch
    import mluop_hip
    rows = 4099
    g = torch.Generator(device="cuda").manual_seed(channels)
    x, dy = (torch.randn(rows, channels, device="cuda", generator=g).to(getattr(torch, dtype)) for _ in range(2))
    w, b = 1 + 0.2 * torch.randn(channels, device="cuda", generator=g), torch.randn(channels, device="cuda", generator=g)
    # (an eps of the spread's size: the root of a row of two values that are almost one hides no error)
    out, mean, rstd = mluop_hip.layer_norm_forward(gpu_handle, x, w, b, 0.1)
    # (on the host: torch's sums of many rows on the GPU by several workgroups have been off)
    leaves = [t.double().cpu().requires_grad_() for t in (x, w, b)]
    want = torch.nn.functional.layer_norm(leaves[0], (channels,), leaves[1], leaves[2], 0.1)
    grads = torch.autograd.grad(want, leaves, dy.double().cpu())
    # a row's sums have at most 48 terms of 2^-24 each, its gradient three such sums of values below 2^6
    row = 160 * 2.0 ** -24
    assert bool(((out.double().cpu() - want).abs() <= LAST[dtype] * want.abs() + row * 8).all())
    got = [t.double().cpu() for t in mluop_hip.layer_norm_backward(gpu_handle, dy, x, w, b, mean, rstd)]
    assert bool(((got[0] - grads[0]).abs() <= LAST[dtype] * grads[0].abs() + row * 64).all())
    # a column: up to 256 teams one after the other, some tens of workgroups, 64 shares, of values below 2^5
    normed = (leaves[0].detach() - mean.double().cpu()[:, None]) * rstd.double().cpu()[:, None]
    for a, c, terms in ((got[1], grads[1], dy.double().cpu() * normed), (got[2], grads[2], dy.double().cpu())):
        assert bool(((a - c).abs() <= 512 * 2.0 ** -24 * terms.abs().sum(0) + rows * row).all())


@pytest.mark.parametrize("dtype", ["float32", "float16"])
@pytest.mark.parametrize("channels", CHANNELS)
@pytest.mark.parametrize("choices", [1, 2, 5])
def test_rows_by_expert(gpu_handle, dtype, channels, choices):
    import torch
    import mluop_hip
    rows, experts = 3001, 11
    chosen, g = routing(rows, choices, experts, channels)
    x, y, dy = (torch.randn(n, channels, device="cuda", generator=g).to(getattr(torch, dtype))
                for n in (rows, rows * choices, rows))
    w = torch.rand(rows, choices, device="cuda", generator=g)
    named, starts, places = mluop_hip.expert_order(gpu_handle, chosen, experts)
    assert torch.equal(mluop_hip.expert_dispatch(gpu_handle, x, places, starts),
                       mluop_hip.embedding_forward(gpu_handle, x, named))

    def near(got, want, size, units, last):
        assert bool(((got.double() - want).abs() <= LAST[last] * want.abs() + units * 2.0 ** -24 * size + LEAST).all())
    terms = taken(y, places) * w.double().unsqueeze(2)
    near(mluop_hip.expert_combine(gpu_handle, y, places, w), terms.sum(dim=1), terms.abs().sum(dim=1), choices + 1, dtype)
    dr, dw = mluop_hip.expert_combine_backward(gpu_handle, dy, y, places, w, starts)
    want, there = torch.zeros(rows * choices, channels, device="cuda", dtype=torch.float64), places >= 0
    want[places[there].long()] = (dy.double().unsqueeze(1) * w.double().unsqueeze(2))[there]
    near(dr, want, want.abs(), 1, dtype)
    terms = dy.double().unsqueeze(1) * taken(y, places)
    near(dw, terms.sum(dim=2), terms.abs().sum(dim=2), channels + 8, "float32")


RAGGED = [3, 3, 4100, 4101, 8900]


@pytest.mark.parametrize("dtype,kind,reverse", [("float32", "sigmoid", False), ("bfloat16", "exp", True),
                                                ("bfloat16", "sigmoid", True), ("float16", "exp", False)])
@pytest.mark.parametrize("rows,starts", [(100, None), (3000, None), (9001, None), (9001, RAGGED), (70, list(range(71)))])
@pytest.mark.parametrize("channels", [1, 3, 8, 12, 16, 20, 32])
def test_recurrence(gpu_handle, dtype, kind, reverse, rows, starts, channels):
    """as whole samples, with tiles that every wave folds, and joined; 4, 8 or 16 lanes across"""
    import torch
    from test_gpu_gated_scan import check, inputs
    samples = 1 if starts is None else len(starts) - 1
    x, g, h0, dh, df = inputs(rows, channels, samples, getattr(torch, dtype), kind, rows + channels)
    check(gpu_handle, x, g, starts, h0, dh, df, kind, reverse, dtype)


@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("rows", [200, 9000])
def test_recurrence_whose_gradients_lie_otherwise(gpu_handle, rows, reverse):
    """a gradient whose rows lie apart at odd places is taken by more lanes than the forward pass's rows were"""
    import torch
    import mluop_hip
    g = torch.Generator(device="cuda").manual_seed(rows)
    x, gates = (torch.randn(rows, 16, device="cuda", generator=g).bfloat16() for _ in range(2))
    wide = torch.randn(rows, 19, device="cuda", generator=g).bfloat16()
    starts = torch.tensor([0, 5, rows - 3], dtype=torch.int32, device="cuda")
    out, final, carries = mluop_hip.gated_scan_forward(gpu_handle, x, gates, starts, reverse=reverse)
    near = mluop_hip.gated_scan_backward(gpu_handle, wide[:, 1:17].contiguous(), None, x, gates, carries, starts, reverse=reverse)
    apart = mluop_hip.gated_scan_backward(gpu_handle, wide[:, 1:17], None, x, gates, carries, starts, reverse=reverse)
    for a, b in zip(near, apart):
        # (the same but for the order of compositions: a rounding to bfloat16 of each, and fp32 sums of values below 2^5)
        assert torch.allclose(a.float(), b.float(), rtol=2.0 ** -7, atol=2.0 ** -14)
    again = mluop_hip.gated_scan_forward(gpu_handle, wide[:, :16], gates, starts, reverse=reverse)
    same = mluop_hip.gated_scan_forward(gpu_handle, wide[:, :16].contiguous(), gates, starts, reverse=reverse)
    for a, b in zip(again[:2], same[:2]):   # (of the carries some rows belong to no sample)
        assert torch.allclose(a.float(), b.float(), rtol=2.0 ** -7, atol=2.0 ** -14)


def lengths(which):
    """of samples: long ones, some of several tiles, and many of few rows or none"""
    import random
    draw = random.Random(which)
    if which == "joined":
        some = [5000, 0, 2500, 700, 64, 65, 128, 129, 1, 256, 257, 300] + [draw.choice([0, 0, 1, 2, 7, 40]) for _ in range(190)]
    elif which == "folded":
        some = [400, 0, 200] + [draw.choice([0, 0, 1, 2, 3, 70]) for _ in range(130)]
    else:
        some = [90, 0] + [draw.choice([0, 0, 1, 1, 2]) for _ in range(170)]
    draw.shuffle(some)
    return some


@pytest.mark.parametrize("dtype,kind,reverse", [("float32", "exp", False), ("bfloat16", "sigmoid", True),
                                                ("float32", "sigmoid", True), ("float16", "exp", False)])
@pytest.mark.parametrize("which", ["whole", "folded", "joined"])
@pytest.mark.parametrize("channels", [5, 12, 72])
def test_recurrence_of_samples_long_and_short(gpu_handle, dtype, kind, reverse, which, channels):
    import torch
    from itertools import accumulate
    from test_gpu_gated_scan import check, inputs
    some = lengths(which)
    starts = [3] + [3 + n for n in accumulate(some)]
    rows = starts[-1] + 2
    x, g, h0, dh, df = inputs(rows, channels, len(some), getattr(torch, dtype), kind, rows + channels)
    check(gpu_handle, x, g, starts, h0, dh, df, kind, reverse, dtype)
