"""Layer norm: values and gradients against float64 at every team and vector width, rows far off zero, constant ones, rows that
are not finite, rows that lie apart; captured graphs; refusals."""
import pytest

pytestmark = pytest.mark.gpu

# One rounding of a result of each type.
LAST = {"float32": 2.0 ** -24, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}
# A sum of a row in fp32 has up to 32 terms of a thread one after the other, then a tree of up to 6 + 16 additions; what is made of
# it some ten roundings more.
ROW = 64 * 2.0 ** -24
LEAST = 2.0 ** -25   # half a step of the smallest numbers of fp16


def inputs(rows, channels, dtype, params, seed, offset=2.0):
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = (torch.randn(rows, channels, device="cuda", generator=g) +
         offset * torch.randn(rows, 1, device="cuda", generator=g)).to(dtype)
    w = (1 + 0.3 * torch.randn(channels, device="cuda", generator=g)).to(params)
    b = (0.3 * torch.randn(channels, device="cuda", generator=g)).to(params)
    dy = torch.randn(rows, channels, device="cuda", generator=g).to(dtype)
    return x, w, b, dy


def forward(x, w, b, eps):
    x = x.double()
    mean = x.mean(dim=1)
    rstd = ((x - mean[:, None]).square().mean(dim=1) + eps) ** -0.5
    y = (x - mean[:, None]) * rstd[:, None]
    if w is not None:
        y = y * w.double()
    return (y if b is None else y + b.double()), mean, rstd


def within(got, want, room):
    import torch
    off = (got.double() - want).abs()
    assert bool((off <= room).all()), float((off / room).max())
    assert not bool(torch.isnan(got).any())


CASES = [(1, 1), (7, 1), (1, 8), (3, 7), (65, 33), (1000, 64), (3001, 64), (517, 100), (300, 128), (120, 250), (90, 257),
         (64, 512), (200, 1000), (40, 1025), (33, 1024), (70, 2048), (21, 2050), (9, 4096), (1, 5000), (5, 8191), (12, 8192),
         (3, 8200), (40, 16384), (2, 32767), (3, 32768), (20000, 16)]


@pytest.mark.parametrize("dtype,params", [("float32", "float32"), ("float16", "float32"), ("bfloat16", "bfloat16")])
@pytest.mark.parametrize("rows,channels", CASES)
def test_against_float64(gpu_handle, dtype, params, rows, channels):
    import torch
    import mluop_hip
    print("layer norm", dtype, params, rows, channels, flush=True)
    x, w, b, dy = inputs(rows, channels, getattr(torch, dtype), getattr(torch, params), rows + channels)
    out, mean, rstd = mluop_hip.layer_norm_forward(gpu_handle, x, w, b, 1e-5)
    want, want_mean, want_rstd = forward(x, w, b, 1e-5)
    # (differences from the mean are off by what the sum of the differences is, and by the mean's last place)
    size = (x.double() - want_mean[:, None]).abs().max(dim=1).values
    within(mean, want_mean, 2.0 ** -23 * want_mean.abs() + ROW * size + 2.0 ** -60)
    # (a row of one channel has no spread: its root is that of eps)
    within(rstd, want_rstd, want_rstd * (ROW + ROW * (size * want_rstd).square()))
    normed = ((x.double() - want_mean[:, None]) * want_rstd[:, None]).abs()
    normed_room = ROW * (1 + (size * want_rstd)[:, None]) * (1 + normed)
    wide = w.double().abs()
    within(out, want, LAST[dtype] * want.abs() + normed_room * wide + 2.0 ** -23 * b.double().abs() + LEAST)

    dx, dw, db = mluop_hip.layer_norm_backward(gpu_handle, dy, x, w, b, mean, rstd)
    m, r, g = mean.double()[:, None], rstd.double()[:, None], dy.double()
    n = (x.double() - m) * r
    d = g * w.double()
    a, c = d.mean(dim=1, keepdim=True), (d * n).mean(dim=1, keepdim=True)
    sizes = d.abs() + d.abs().mean(dim=1, keepdim=True) + n.abs() * (d * n).abs().mean(dim=1, keepdim=True)
    within(dx, r * (d - a - n * c), LAST[dtype] * (r * (d - a - n * c)).abs() + ROW * r * sizes + LEAST)
    # sums down the columns: a thread's rows one after the other (up to 40 here), its workgroup's 32 teams, 32 parts, 16 shares
    column = 160 * 2.0 ** -24
    for got, terms in ((dw, g * n), (db, g)):
        # (on the host: torch's sums of many rows on the GPU by several workgroups have been off)
        total, sizes = terms.cpu().sum(dim=0).cuda(), terms.cpu().abs().sum(dim=0).cuda()
        within(got, total, LAST[params] * total.abs() + column * sizes + LEAST)


def test_gradient_by_differences(gpu_handle):
    import torch
    import mluop_hip
    x, w, b, dy = inputs(13, 24, torch.float32, torch.float32, 5, offset=0.5)
    out, mean, rstd = mluop_hip.layer_norm_forward(gpu_handle, x, w, b)
    grads = mluop_hip.layer_norm_backward(gpu_handle, dy, x, w, b, mean, rstd)
    g = torch.Generator(device="cuda").manual_seed(0)
    for k, t in enumerate((x, w, b)):
        for _ in range(4):
            # (central differences of h = 2^-10 in float64 of the definition: off by h^2 of its third derivative)
            d, h = torch.randn(t.shape, device="cuda", generator=g).double(), 2.0 ** -10
            values = []
            for s in (1, -1):
                args = [v.double() for v in (x, w, b)]
                args[k] = args[k] + s * h * d
                values.append(float((forward(*args, 1e-5)[0] * dy.double()).sum()))
            slope, want = (values[0] - values[1]) / (2 * h), float((grads[k].double() * d).sum())
            assert abs(slope - want) <= 1e-4 * (abs(want) + float(d.norm()))


@pytest.mark.parametrize("weight,bias", [(False, False), (True, False), (False, True)])
def test_without_weight_or_bias(gpu_handle, weight, bias):
    import torch
    import mluop_hip
    from mluop_hip import nn as spnn
    x, w, b, dy = inputs(77, 96, torch.float32, torch.float32, 8)
    w, b = (w if weight else None), (b if bias else None)
    out, mean, rstd = mluop_hip.layer_norm_forward(gpu_handle, x, w, b)
    within(out, forward(x, w, b, 1e-5)[0], 64 * 2.0 ** -20)
    leaves = [t.clone().requires_grad_() for t in (x, w, b) if t is not None]
    args = iter(leaves)
    y = spnn.layer_norm(next(args), next(args) if weight else None, next(args) if bias else None)
    assert torch.equal(y, out)
    have = torch.autograd.grad(y, leaves, dy)
    want = [g for g, t in zip(mluop_hip.layer_norm_backward(gpu_handle, dy, x, w, b, mean, rstd), (x, w, b)) if t is not None]
    assert all(torch.equal(a, c) for a, c in zip(have, want))
    # (the last of them alone)
    leaf = leaves[-1].detach().clone().requires_grad_()
    rest = iter([t.detach() for t in leaves[:-1]] + [leaf])
    y = spnn.layer_norm(next(rest), next(rest) if weight else None, next(rest) if bias else None)
    assert torch.equal(torch.autograd.grad(y, leaf, dy)[0], want[-1])


def test_rows_far_off_zero_and_constant_ones(gpu_handle):
    import torch
    import mluop_hip
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(50, 256, device="cuda", generator=g) + 3000.0
    x[25:] = 7.25
    out, mean, rstd = mluop_hip.layer_norm_forward(gpu_handle, x, None, None)
    want, want_mean, want_rstd = forward(x, None, None, 1e-5)
    # (no more is lost than the mean's own last place, which is 2^-13 of a spread)
    assert bool(((mean.double() - want_mean).abs() <= 2.0 ** -23 * want_mean.abs()).all())
    assert bool(((rstd.double() / want_rstd - 1).abs() <= 64 * 2.0 ** -24).all())
    assert float((out.double() - want).abs().max()) <= 2.0 ** -17
    assert not bool(out[25:].any())


def test_rows_that_are_not_finite_stay_by_themselves(gpu_handle):
    import torch
    import mluop_hip
    for channels in (64, 1000, 9000):
        x, w, b, dy = inputs(20, channels, torch.float16, torch.float32, 2)
        clean, mean, rstd = mluop_hip.layer_norm_forward(gpu_handle, x, w, b)
        x2 = x.clone()
        x2[3, 5], x2[17, 60] = float("inf"), float("nan")
        out, mean, rstd = mluop_hip.layer_norm_forward(gpu_handle, x2, w, b)
        bad = torch.zeros(20, dtype=torch.bool, device="cuda")
        bad[[3, 17]] = True
        assert torch.equal(out[~bad], clean[~bad]) and bool(torch.isnan(out[bad]).all())
        dx = mluop_hip.layer_norm_backward(gpu_handle, dy, x2, w, b, mean, rstd)[0]
        assert bool(torch.isnan(dx[bad]).all()) and bool(torch.isfinite(dx[~bad]).all())


def test_rows_apart_and_unaligned(gpu_handle):
    """views: every second row, columns of a wider tensor, addresses that no vector load takes, transposed and expanded ones"""
    import torch
    import mluop_hip
    x, w, b, dy = inputs(200, 64, torch.float16, torch.float16, 9)
    want = mluop_hip.layer_norm_forward(gpu_handle, x, w, b)
    grads = mluop_hip.layer_norm_backward(gpu_handle, dy, x, w, b, *want[1:])
    wide = torch.zeros(400, 160, dtype=torch.float16, device="cuda")
    flat = torch.zeros(200 * 64 + 1, dtype=torch.float16, device="cuda")
    for view in (wide[::2, 16:80], wide[::2, 3:67], flat[1:].view(200, 64), torch.empty(64, 200, dtype=torch.float16, device="cuda").t()):
        view.copy_(x)
        got = mluop_hip.layer_norm_forward(gpu_handle, view, w, b)
        for a, c in zip(got, want):
            assert torch.allclose(a.float(), c.float(), rtol=2.0 ** -10, atol=2.0 ** -18)
        view.copy_(dy)
        for a, c in zip(mluop_hip.layer_norm_backward(gpu_handle, view, x, w, b, *want[1:]), grads):
            assert torch.allclose(a.float(), c.float(), rtol=2.0 ** -9, atol=2.0 ** -12)
    one = x[:1].expand(200, 64)
    assert torch.equal(mluop_hip.layer_norm_forward(gpu_handle, one, w, b)[0], want[0][:1].expand(200, 64))
    params = torch.zeros(3 * 64 + 1, dtype=torch.float16, device="cuda")[1::3]   # (parameters that lie apart)
    params.copy_(w)
    assert torch.equal(mluop_hip.layer_norm_forward(gpu_handle, x, params, b)[0], want[0])


def test_no_rows(gpu_handle):
    import torch
    import mluop_hip
    x, w = torch.zeros(0, 40, device="cuda"), torch.ones(40, device="cuda")
    out, mean, rstd = mluop_hip.layer_norm_forward(gpu_handle, x, w, w)
    assert out.shape == (0, 40) and mean.shape == rstd.shape == (0,)
    dx, dw, db = mluop_hip.layer_norm_backward(gpu_handle, x, x, w, w, mean, rstd)
    assert dx.shape == (0, 40) and not bool(dw.any()) and not bool(db.any())


def test_module_on_sparse_and_higher_tensors():
    import torch
    from mluop_hip import nn as spnn
    layer = spnn.LayerNorm(32).cuda()
    torch.nn.init.normal_(layer.weight)
    x = torch.randn(3, 5, 32, device="cuda", requires_grad=True)
    y = layer(x)
    assert y.shape == x.shape
    assert torch.allclose(y, torch.nn.functional.layer_norm(x, (32,), layer.weight, layer.bias), atol=1e-5)
    y.square().sum().backward()
    idx = torch.tensor([[0, 0, i // 5, i % 5] for i in range(15)], dtype=torch.int32, device="cuda")
    net = spnn.SparseSequential(spnn.SubMConv3d(32, 32, 3), layer).cuda()
    out = net(spnn.SparseTensor(x.detach().view(15, 32), idx, (1, 5, 5), 1, distinct=True))
    assert torch.allclose(out.features, layer(net[0](spnn.SparseTensor(x.detach().view(15, 32), idx, (1, 5, 5), 1)).features),
                          atol=1e-5)


@pytest.mark.parametrize("channels", [48, 2048, 10240])
def test_captured_with_its_gradients(channels):
    import torch
    from mluop_hip import nn as spnn
    x, w, b, dy = inputs(300, channels, torch.bfloat16, torch.float32, 3)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())

    def step():
        leaves = [t.detach().requires_grad_() for t in (x, w, b)]
        y = spnn.layer_norm(*leaves)
        return [y] + list(torch.autograd.grad(y, leaves, dy))
    with torch.cuda.stream(stream):
        step()
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            out = step()
    torch.cuda.synchronize()
    for _ in range(3):
        x.copy_(torch.randn_like(x))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, c) for a, c in zip(out, step()))


def test_refusals(gpu_handle):
    import torch
    import mluop_hip
    x, w, b, dy = inputs(10, 8, torch.float16, torch.float32, 1)
    f = mluop_hip.layer_norm_forward
    for bad in (dict(features=x.double()), dict(features=x[0]), dict(features=x[:, :0]), dict(features=x.cpu()),
                dict(weight=w[:4]), dict(weight=w.half()), dict(bias=b.double()), dict(weight=w.cpu())):
        with pytest.raises(ValueError):
            f(gpu_handle, **{**dict(features=x, weight=w, bias=b), **bad})
    for eps in (-1.0, float("nan"), float("inf")):
        with pytest.raises(mluop_hip.MluOpError):
            f(gpu_handle, x, w, b, eps)
    with pytest.raises(mluop_hip.MluOpError):
        f(gpu_handle, torch.zeros(1, 40000, device="cuda"), None, None)
    out, mean, rstd = f(gpu_handle, x, w, b)
    for bad in (dict(mean=mean.half()), dict(rstd=rstd[:4]), dict(output_grad=dy[:5]), dict(output_grad=dy.float())):
        with pytest.raises(ValueError):
            mluop_hip.layer_norm_backward(gpu_handle, **{**dict(output_grad=dy, features=x, weight=w, bias=b, mean=mean,
                                                                rstd=rstd), **bad})
