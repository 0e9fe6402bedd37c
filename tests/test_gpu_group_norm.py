"""Group norm with an activation over ragged samples: values and gradients against float64 at every vector width, samples of
no rows and of one, rows outside of all samples, channels far off zero, constant channels; the layer on a SparseTensor."""
import pytest

pytestmark = pytest.mark.gpu

# One rounding of a result of each type; what fp32 sums of n terms may be off is added by the tests.
LAST = {"float32": 2.0 ** -24, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}


def reference(x, w, b, groups, starts, eps, act, dy=None):
    """(out, mean, rstd) or gradients by autograd, in float64 on the CPU"""
    import torch
    x = x.detach().double().cpu().requires_grad_()
    w = (torch.ones(x.shape[1]) if w is None else w.detach()).double().cpu().requires_grad_()
    b = (torch.zeros(x.shape[1]) if b is None else b.detach()).double().cpu().requires_grad_()
    out, means, rstds = torch.zeros_like(x), [], []
    parts = []
    for lo, hi in zip(starts, starts[1:]):
        v = x[lo:hi].reshape(hi - lo, groups, x.shape[1] // groups)
        if hi == lo:
            means.append(torch.zeros(groups, dtype=torch.float64))
            rstds.append(torch.full((groups,), eps, dtype=torch.float64) ** -0.5)
            parts.append(x[lo:hi])
            continue
        mean = v.mean(dim=(0, 2))
        rstd = (v.var(dim=(0, 2), unbiased=False) + eps) ** -0.5
        z = ((v - mean[None, :, None]) * rstd[None, :, None]).reshape(hi - lo, -1) * w + b
        parts.append(torch.relu(z) if act == "relu" else z * torch.sigmoid(z) if act == "silu" else z)
        means.append(mean)
        rstds.append(rstd)
    out = torch.cat([torch.zeros_like(x[:starts[0]])] + parts + [torch.zeros_like(x[starts[-1]:])])
    if dy is None:
        return out.detach(), torch.stack(means).detach(), torch.stack(rstds).detach()
    return torch.autograd.grad(out, (x, w, b), dy.detach().double().cpu(), allow_unused=True)


def inputs(rows, channels, dtype, params, seed, offset=2.0):
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = (torch.randn(rows, channels, device="cuda", generator=g) +
         offset * torch.randn(channels, device="cuda", generator=g)).to(dtype)
    w = (1 + 0.3 * torch.randn(channels, device="cuda", generator=g)).to(params)
    b = (0.3 * torch.randn(channels, device="cuda", generator=g)).to(params)
    dy = torch.randn(rows, channels, device="cuda", generator=g).to(dtype)
    return x, w, b, dy


def near(got, want, last, room):
    import torch
    want = want.to(got.device)
    off = (got.double() - want).abs()
    allowed = last * want.abs() + room
    assert bool((off <= allowed).all()), float((off / allowed).max())
    assert not bool(torch.isnan(got).any())


CASES = [  # rows, channels, groups, starts
    (1, 1, 1, None), (1, 8, 2, None), (3, 7, 7, None), (65, 33, 3, [0, 30, 65]), (1000, 64, 16, [0, 0, 1, 1000, 1000]),
    (3001, 64, 32, None), (2500, 20, 5, [7, 1200, 2400]), (700, 128, 32, [0, 100, 700]), (40, 4104, 8, [0, 17, 40]),
    (30, 2056, 257, None), (5000, 4, 1, [0, 2000, 5000]), (6000, 2, 2, [0, 5999, 6000]), (513, 48, 16, list(range(0, 514, 3)))]


@pytest.mark.parametrize("dtype,params", [("float32", "float32"), ("float16", "float32"), ("bfloat16", "bfloat16")])
@pytest.mark.parametrize("act", ["none", "relu", "silu"])
@pytest.mark.parametrize("rows,channels,groups,starts", CASES)
def test_against_float64(gpu_handle, dtype, params, act, rows, channels, groups, starts):
    import torch
    import mluop_hip
    print("group norm", dtype, params, act, rows, channels, groups, flush=True)
    x, w, b, dy = inputs(rows, channels, getattr(torch, dtype), getattr(torch, params), rows + channels)
    host = starts or [0, rows]
    dev = None if starts is None else torch.tensor(starts, dtype=torch.int32, device="cuda")
    out, mean, rstd = mluop_hip.group_norm_forward(gpu_handle, x, w, b, groups, dev, 1e-5, act)
    ref, ref_mean, ref_rstd = reference(x, w, b, groups, host, 1e-5, act)
    # sums of up to a thousand terms in a row, then a tree: a relative 2^-18 of the magnitudes they add up
    size = float(x.float().abs().max())
    # (of samples that have rows)
    spread = ref_rstd[[hi > lo for lo, hi in zip(host, host[1:])]].max().item()
    near(mean, ref_mean, 0, 2.0 ** -20 * size)
    near(rstd, ref_rstd, 2.0 ** -16 * min(1.0 + size * size * 1e-2, 100.0), 0)
    z = 2.0 ** -18 * (1 + size * spread) * float(w.float().abs().max())
    near(out, ref, LAST[dtype] + 2.0 ** -15, 4 * z + 2.0 ** -25)
    # backward from the moments the forward call gave
    got = mluop_hip.group_norm_backward(gpu_handle, dy, x, w, b, mean, rstd, groups, dev, act)
    want = reference(x, w, b, groups, host, 1e-5, act, dy)
    if act == "relu":   # a value within rounding of zero may fall on either side
        zs = reference(x, w, b, groups, host, 1e-5, "none")[0]
        unsure = (zs.abs() <= 8 * z).to("cuda")
        assert float(unsure.float().mean()) < 0.05 or rows * channels < 200
    else:
        unsure = torch.zeros_like(x, dtype=torch.bool)
    scale = float(want[0].abs().max())
    most = float(dy.float().abs().max()) * float(w.float().abs().max())
    clear = ~unsure
    slack = 2.0 ** -15 * (scale + spread * most) + float(unsure.any()) * 0.2 * spread * most
    near(torch.where(clear, got[0], torch.zeros_like(got[0])), want[0] * clear.cpu(), LAST[dtype] + 2.0 ** -14, slack)
    last = LAST[params]
    normed = 2.0 ** -15 * rows * most * (1 + size * spread) / max(1.0, rows ** 0.5)
    doubt = unsure.sum(dim=0).max().item() * 8.0
    near(got[1], want[1], last + 2.0 ** -15, normed + doubt * most)
    near(got[2], want[2], last + 2.0 ** -15, normed + doubt)


def test_gradient_against_differences(gpu_handle):
    import torch
    import mluop_hip
    starts = torch.tensor([0, 9, 31], dtype=torch.int32, device="cuda")
    x, w, b, dy = inputs(31, 12, torch.float32, torch.float32, 4, offset=0.5)

    def value(x, w, b):
        out = mluop_hip.group_norm_forward(gpu_handle, x, w, b, 4, starts, 1e-5, "silu")[0]
        return float((out.double() * dy.double()).sum())
    _, mean, rstd = mluop_hip.group_norm_forward(gpu_handle, x, w, b, 4, starts, 1e-5, "silu")
    grads = mluop_hip.group_norm_backward(gpu_handle, dy, x, w, b, mean, rstd, 4, starts, "silu")
    g = torch.Generator(device="cuda").manual_seed(0)
    for k, t in enumerate((x, w, b)):
        for _ in range(4):
            # along a direction: second-order differences of h = 1/64 are off by h^2, the values by fp32 roundings
            d = torch.randn(t.shape, device="cuda", generator=g)
            h = 1.0 / 64
            args = [[x, w, b], [x, w, b]]
            args[0][k], args[1][k] = t + h * d, t - h * d
            slope = (value(*args[0]) - value(*args[1])) / (2 * h)
            want = float((grads[k].double() * d.double()).sum())
            assert abs(slope - want) <= 0.02 * (abs(want) + float(d.norm()))


def test_channels_far_off_zero_and_constant_ones(gpu_handle):
    """mean / spread of 3000: a variance from sums of squares in fp32 would be lost"""
    import torch
    import mluop_hip
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(20000, 8, device="cuda", generator=g) + 3000.0
    x[:, 4:] = 7.25
    out, mean, rstd = mluop_hip.group_norm_forward(gpu_handle, x, None, None, 2)
    ref, ref_mean, ref_rstd = reference(x, None, None, 2, [0, 20000], 1e-5, "none")
    assert bool(((mean.cpu().double() - ref_mean).abs() <= 2.0 ** -22 * ref_mean.abs()).all())
    # (the values themselves have a unit of 2^-12 in their last place)
    assert bool(((rstd.cpu().double() / ref_rstd - 1).abs() <= 1e-5).all())
    assert bool((out[:, 4:] == 0).all())
    assert float((out.cpu().double() - ref).abs().max()) <= 2.0 ** -10
    x[0, 0] = -2e6   # a first row that is far from all others
    rstd = mluop_hip.group_norm_forward(gpu_handle, x, None, None, 2)[2]
    ref_rstd = reference(x, None, None, 2, [0, 20000], 1e-5, "none")[2]
    assert bool(((rstd.cpu().double() / ref_rstd - 1).abs() <= 1e-4).all())


def test_rows_that_are_not_finite_stay_in_their_sample(gpu_handle):
    import torch
    import mluop_hip
    x, w, b, dy = inputs(300, 16, torch.float16, torch.float32, 2)
    starts = torch.tensor([0, 100, 200, 300], dtype=torch.int32, device="cuda")
    clean = mluop_hip.group_norm_forward(gpu_handle, x, w, b, 4, starts, 1e-5, "silu")
    x2 = x.clone()
    x2[150, 3], x2[160, 9] = float("inf"), float("nan")
    out, mean, rstd = mluop_hip.group_norm_forward(gpu_handle, x2, w, b, 4, starts, 1e-5, "silu")
    for lo, hi in ((0, 100), (200, 300)):
        assert torch.equal(out[lo:hi], clean[0][lo:hi])
    assert torch.equal(out[100:200, 4:8], clean[0][100:200, 4:8])   # (another group)
    assert bool(torch.isnan(out[100:200, 8:12]).all()) and not bool(torch.isfinite(mean[1, 0]))


def test_no_rows(gpu_handle):
    import torch
    import mluop_hip
    x = torch.zeros(0, 8, device="cuda")
    w = torch.ones(8, device="cuda")
    out, mean, rstd = mluop_hip.group_norm_forward(gpu_handle, x, w, w, 2, None, 0.25)
    assert out.shape == (0, 8) and not bool(mean.any()) and bool((rstd == 2.0).all())
    dx, dw, db = mluop_hip.group_norm_backward(gpu_handle, x, x, w, w, mean, rstd, 2)
    assert dx.shape == (0, 8) and not bool(dw.any()) and not bool(db.any())


def test_starts_that_make_no_sense_stay_in_bounds(gpu_handle):
    """(their results are undefined; no access leaves a tensor: outputs lie between guard bands)"""
    import torch
    import mluop_hip
    x, w, b, dy = inputs(3000, 16, torch.float16, torch.float32, 2)
    for starts in ([0, 3000, 0, 3000, 0, 3000], [-7, 1 << 30, 5, 4, 3, 2], [9] * 6, [3000, 0, -1, 3000, 0, 1]):
        dev = torch.tensor(starts, dtype=torch.int32, device="cuda")
        out, mean, rstd = mluop_hip.group_norm_forward(gpu_handle, x, w, b, 4, dev)
        mluop_hip.group_norm_backward(gpu_handle, dy, x, w, b, mean, rstd, 4, dev)
    torch.cuda.synchronize()


def test_rows_apart_and_unaligned(gpu_handle):
    """views: every second row, columns of a wider tensor, an address that no vector load takes"""
    import torch
    import mluop_hip
    x, w, b, dy = inputs(200, 16, torch.float16, torch.float16, 9)
    want = mluop_hip.group_norm_forward(gpu_handle, x, w, b, 4, None, 1e-5, "relu")
    wide = torch.zeros(400, 40, dtype=torch.float16, device="cuda")
    wide[::2, 3:19] = x
    flat = torch.zeros(200 * 16 + 1, dtype=torch.float16, device="cuda")
    flat[1:] = x.flatten()
    for view in (wide[::2, 3:19], flat[1:].view(200, 16)):
        got = mluop_hip.group_norm_forward(gpu_handle, view, w, b, 4, None, 1e-5, "relu")
        assert float((got[0] - want[0]).abs().max()) <= 2.0 ** -8 and torch.allclose(got[1], want[1], atol=1e-6)


def test_layer_and_autograd():
    import torch
    from mluop_hip import nn as spnn
    torch.manual_seed(1)
    idx = torch.tensor([[n, 0, i // 20, i % 20] for n in range(3) for i in range(60 + 50 * n)], dtype=torch.int32,
                       device="cuda")
    feats = torch.randn(idx.shape[0], 16, device="cuda", requires_grad=True)
    net = spnn.SparseSequential(spnn.SubMConv3d(16, 32, 3), spnn.GroupNormAct(8, 32, activation="silu"),
                                spnn.SubMConv3d(32, 32, 3)).cuda()
    x = spnn.SparseTensor(feats, idx, (1, 20, 20), 3, distinct=True)
    y = net(x)
    mid = net[0](x).features
    starts = [0, 60, 170, 330]
    assert x.row_starts().tolist() == starts
    ref = torch.cat([torch.nn.functional.silu(torch.nn.functional.group_norm(
        mid[a:b].t()[None], 8, net[1].weight, net[1].bias, 1e-5))[0].t() for a, b in zip(starts, starts[1:])])
    got = net[1](net[0](x)).features
    assert torch.allclose(got, ref, atol=1e-5)
    want = torch.autograd.grad((ref * torch.arange(32.0, device="cuda")).sum(), [feats, net[1].weight, net[1].bias],
                               retain_graph=True)
    have = torch.autograd.grad((got * torch.arange(32.0, device="cuda")).sum(), [feats, net[1].weight, net[1].bias])
    for a, b in zip(have, want):
        assert torch.allclose(a, b, rtol=1e-3, atol=1e-3 * float(b.abs().max()))
    y.features.square().mean().backward()
    assert all(p.grad is not None for p in net.parameters())


def test_captured_and_on_another_stream():
    import torch
    from mluop_hip import nn as spnn
    x, w, b, dy = inputs(5000, 64, torch.float16, torch.float32, 3)
    starts = torch.tensor([0, 2000, 5000], dtype=torch.int32, device="cuda")
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        spnn.group_norm(x, w, b, 16, starts, activation="silu")
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            out = spnn.group_norm(x, w, b, 16, starts, activation="silu")
    torch.cuda.synchronize()
    for k in range(3):
        x.copy_(torch.randn_like(x))
        starts[1] = 1000 + k
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, spnn.group_norm(x, w, b, 16, starts, activation="silu"))


def test_refusals(gpu_handle):
    import torch
    import mluop_hip
    x, w, b, dy = inputs(10, 8, torch.float16, torch.float32, 1)
    f = mluop_hip.group_norm_forward
    starts = torch.tensor([0, 10], dtype=torch.int32, device="cuda")
    for bad in (dict(features=x.double()), dict(features=x[0]), dict(groups=3), dict(groups=0), dict(weight=w[:4]),
                dict(weight=w.half()), dict(bias=b.double()), dict(row_starts=starts.long()), dict(row_starts=starts[:1]),
                dict(row_starts=starts.cpu()), dict(features=x.cpu())):
        with pytest.raises(ValueError):
            f(gpu_handle, **{**dict(features=x, weight=w, bias=b, groups=2, row_starts=starts), **bad})
    with pytest.raises(KeyError):
        f(gpu_handle, x, w, b, 2, activation="gelu")
    with pytest.raises(mluop_hip.MluOpError):
        f(gpu_handle, x, w, b, 2, eps=-1.0)
    out, mean, rstd = f(gpu_handle, x, w, b, 2)
    for bad in (dict(mean=mean.half()), dict(rstd=rstd[:, :1]), dict(output_grad=dy[:5]), dict(output_grad=dy.float())):
        with pytest.raises(ValueError):
            mluop_hip.group_norm_backward(gpu_handle, **{**dict(output_grad=dy, features=x, weight=w, bias=b, mean=mean,
                                                                rstd=rstd, groups=2), **bad})
