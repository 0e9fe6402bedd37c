"""Products grouped by expert: forward and both gradients against float64 at groups of no row, one and many, sizes around
tiles and vectors, rows of no group, strides and addresses that vector loads do not take, values that are not finite in
rows and filters that nobody uses; slices of the filter's gradient; the layer with autograd."""
import pytest

pytestmark = pytest.mark.gpu

LAST = {"float32": 2.0 ** -24, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}


def starts_of(sizes, first=0):
    out = [first]
    for n in sizes:
        out.append(out[-1] + n)
    return out


def inputs(rows, groups, ci, co, dtype, seed):
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(rows, ci, device="cuda", generator=g).to(dtype)
    w = (torch.randn(groups, ci, co, device="cuda", generator=g) * ci ** -0.5).to(dtype)
    dy = torch.randn(rows, co, device="cuda", generator=g).to(dtype)
    return x, w, dy


def reference(x, w, dy, starts):
    """values and sums of magnitudes of the three products, in float64"""
    import torch
    out = []
    x, w, dy = x.double(), w.double(), dy.double()
    for f in (lambda t: t, torch.abs):
        y, dx, dw = torch.zeros_like(dy), torch.zeros_like(x), torch.zeros_like(w)
        for k, (a, b) in enumerate(zip(starts, starts[1:])):
            y[a:b] = f(x[a:b]) @ f(w[k])
            dx[a:b] = f(dy[a:b]) @ f(w[k]).t().contiguous()
            dw[k] = f(x[a:b]).t().contiguous() @ f(dy[a:b])
        out.append((y, dx, dw))
    return out


def products(handle, x, w, dy, dev):
    import mluop_hip
    return (mluop_hip.grouped_matmul_forward(handle, x, w, dev),
            mluop_hip.grouped_matmul_backward_data(handle, dy, w, dev),
            mluop_hip.grouped_matmul_backward_filter(handle, x, dy, dev))


def compare(got, x, w, dy, starts, dtype):
    values, sizes = reference(x, w, dy, starts)
    longest = max([b - a for a, b in zip(starts, starts[1:])] + [1])
    for name, g, v, s, n in zip(("out", "input_grad", "filters_grad"), got, values, sizes,
                                (x.shape[1], dy.shape[1], longest)):
        # n products in any order: each sum rounds by half a unit of what has been added up, products of fp32 once themselves
        # (a matrix instruction may cut instead of round: a whole unit)
        room = (n + 2) * 2.0 ** -23 * s + LAST[dtype] * v.abs() + 2.0 ** -25
        off = (g.double() - v).abs()
        assert bool((off <= room).all()), (name, float((off / room).max()))


SHAPES = [  # sizes of the groups, first row, rows behind the last group, ci, co
    ([1], 0, 0, 1, 1), ([1], 0, 0, 64, 64), ([3, 0, 5], 0, 0, 7, 9), ([0, 0, 0], 0, 0, 16, 16), ([0, 2, 0], 0, 0, 40, 24),
    ([63, 65, 64, 1], 0, 0, 64, 128), ([17, 0, 130], 5, 9, 96, 72), ([200], 3, 0, 33, 65), ([16, 16, 15, 17, 1], 0, 0, 256, 512),
    ([300, 2, 257], 0, 1, 128, 128), ([1, 1, 1, 1, 1, 1, 1, 1], 0, 0, 512, 264), ([129], 0, 0, 1024, 1000),
    ([1000, 31], 0, 0, 136, 264), ([255, 256, 257], 0, 0, 72, 320), ([5000], 0, 0, 48, 40), ([2100, 0, 2100], 7, 7, 16, 32),
    ([2] * 70, 0, 0, 32, 8), ([12, 3, 700, 90], 0, 0, 512, 768)]


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("sizes,first,behind,ci,co", SHAPES)
def test_against_float64(gpu_handle, dtype, sizes, first, behind, ci, co):
    import torch
    print("grouped", dtype, sizes[:8], first, behind, ci, co, flush=True)
    starts = starts_of(sizes, first)
    x, w, dy = inputs(starts[-1] + behind, len(sizes), ci, co, getattr(torch, dtype), ci + co)
    dev = torch.tensor(starts, dtype=torch.int32, device="cuda")
    got = products(gpu_handle, x, w, dy, dev)
    compare(got, x, w, dy, starts, dtype)
    for t in got[:2]:
        assert not bool(t[:first].any()) and not bool(t[starts[-1]:].any())
    again = products(gpu_handle, x, w, dy, dev)
    assert all(torch.equal(a, b) for a, b in zip(got, again))


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("groups,rows,ci,co", [(8, 2600, 512, 1024), (3, 4000, 1000, 520), (24, 1500, 256, 2048)])
def test_larger(gpu_handle, dtype, groups, rows, ci, co):
    import random
    import torch
    print("grouped larger", dtype, groups, rows, ci, co, flush=True)
    rng = random.Random(rows)
    cuts = sorted(rng.randrange(rows + 1) for _ in range(groups - 1))
    starts = [0] + cuts + [rows]
    x, w, dy = inputs(rows, groups, ci, co, getattr(torch, dtype), 3)
    dev = torch.tensor(starts, dtype=torch.int32, device="cuda")
    compare(products(gpu_handle, x, w, dy, dev), x, w, dy, starts, dtype)


def launched(handle, call):
    """(the call's result, the names of the kernels it launched)"""
    import mluop_hip
    handle.set_kernel_timing(True)
    try:
        out = call()
        return out, [name for name, _ in handle.kernel_timings()]
    finally:
        handle.set_kernel_timing(False)


KINDS = [  # groups, rows, ci, co, the kernels of the three products
    (3, 40, 512, 1032, ("groupedFew16", "groupedFew16", "groupedTiles")),
    (2, 700, 1024, 520, ("groupedFew", "groupedFew", "groupedTiles")),
    (5, 1200, 2048, 2048, ("groupedFew64x128", "groupedFew64x128", "groupedTiles")),
    (1, 4100, 2056, 2048, ("groupedTiles128", "groupedTiles128", "groupedTiles")),
    (7, 16000, 1032, 1024, ("groupedTiles", "groupedTiles", "groupedTiles")),
    (1, 16000, 2048, 2048, ("groupedTiles256", "groupedTiles256", "groupedTiles256")),
    (1, 30000, 64, 72, ("groupedFew64", "groupedFew64", "groupedTiles"))]


@pytest.mark.parametrize("groups,rows,ci,co,kinds", KINDS)
def test_every_tile(gpu_handle, groups, rows, ci, co, kinds):
    """uneven groups at sizes at which each kernel is the one that runs (small whole numbers: sums are exact in fp32)"""
    import random
    import torch
    import mluop_hip
    print("grouped tiles", groups, rows, ci, co, flush=True)
    g = torch.Generator(device="cuda").manual_seed(rows)
    rng = random.Random(groups)
    starts = [0] + sorted(rng.randrange(rows + 1) for _ in range(groups - 1)) + [rows]
    x = torch.randint(-2, 3, (rows, ci), device="cuda", generator=g).half()
    w = torch.randint(-1, 2, (groups, ci, co), device="cuda", generator=g).half()
    dy = torch.randint(-1, 2, (rows, co), device="cuda", generator=g).half()
    dev = torch.tensor(starts, dtype=torch.int32, device="cuda")
    want = [torch.empty_like(dy, dtype=torch.float32), torch.empty_like(x, dtype=torch.float32),
            torch.empty(w.shape, device="cuda")]
    for k, (a, b) in enumerate(zip(starts, starts[1:])):
        want[0][a:b] = x[a:b].float() @ w[k].float()
        want[1][a:b] = dy[a:b].float() @ w[k].float().t().contiguous()
        want[2][k] = x[a:b].float().t().contiguous() @ dy[a:b].float()
    calls = (lambda: mluop_hip.grouped_matmul_forward(gpu_handle, x, w, dev),
             lambda: mluop_hip.grouped_matmul_backward_data(gpu_handle, dy, w, dev),
             lambda: mluop_hip.grouped_matmul_backward_filter(gpu_handle, x, dy, dev))
    for call, v, kind in zip(calls, want, kinds):
        got, names = launched(gpu_handle, call)
        assert names and names[0].startswith(kind), names
        assert float(v.abs().max()) < 2 ** 24 and torch.equal(got, v.half())


def test_integers_are_exact(gpu_handle):
    """small whole numbers: every sum is exact in fp32, so any wrong element shows"""
    import torch
    g = torch.Generator(device="cuda").manual_seed(1)
    sizes, ci, co = [70, 0, 300, 129, 1], 264, 392
    starts = starts_of(sizes)
    x = torch.randint(-3, 4, (starts[-1], ci), device="cuda", generator=g).to(torch.bfloat16)
    w = torch.randint(-2, 3, (5, ci, co), device="cuda", generator=g).to(torch.bfloat16)
    dy = torch.randint(-3, 4, (starts[-1], co), device="cuda", generator=g).to(torch.bfloat16)
    dev = torch.tensor(starts, dtype=torch.int32, device="cuda")
    got = products(gpu_handle, x, w, dy, dev)
    for g, v in zip(got, reference(x, w, dy, starts)[0]):
        assert torch.equal(g, v.to(torch.bfloat16))


def test_what_nobody_uses_is_not_looked_at(gpu_handle):
    """infinities and NaN in the filter of an empty group, in rows of other groups and of none"""
    import torch
    sizes, first = [40, 0, 90], 10
    starts = starts_of(sizes, first)
    for ci, co in ((64, 128), (72, 40), (33, 17)):
        x, w, dy = inputs(starts[-1] + 10, 3, ci, co, torch.float16, 8)
        dev = torch.tensor(starts, dtype=torch.int32, device="cuda")
        clean = products(gpu_handle, x, w, dy, dev)
        w2, x2, dy2 = w.clone(), x.clone(), dy.clone()
        w2[1] = float("nan")
        for t in (x2, dy2):
            t[:first] = float("inf")
            t[starts[-1]:] = float("nan")
        got = products(gpu_handle, x2, w2, dy2, dev)
        assert all(torch.equal(a, b) for a, b in zip(got, clean))
        assert not bool(got[2][1].any())
        # and a row of one group reaches no other
        x2[starts[0] + 5, 3], dy2[starts[0] + 5, 2] = float("nan"), float("inf")
        w2[0, 1, 1] = float("nan")
        got = products(gpu_handle, x2, w2, dy2, dev)
        for a, b in zip(got[:2], clean[:2]):
            assert torch.equal(a[starts[1]:], b[starts[1]:])
        assert torch.equal(got[2][1:], clean[2][1:])


def test_strides_and_alignment(gpu_handle):
    import torch
    import mluop_hip
    sizes = [30, 50, 0, 20]
    starts = starts_of(sizes)
    x, w, dy = inputs(100, 4, 64, 96, torch.bfloat16, 2)
    dev = torch.tensor(starts, dtype=torch.int32, device="cuda")
    want = products(gpu_handle, x, w, dy, dev)
    wide = torch.zeros(100, 300, dtype=torch.bfloat16, device="cuda")
    for at in (8, 3):
        xv, dyv = wide[:, at:at + 64], wide[:, 100 + at:196 + at]
        xv.copy_(x)
        dyv.copy_(dy)
        for a, b in zip(products(gpu_handle, xv, w, dyv, dev), want):
            assert torch.allclose(a.float(), b.float(), rtol=2.0 ** -7, atol=1e-5 * float(b.float().abs().max()) + 1e-3)
    xt = x.t().contiguous().t()
    assert torch.equal(mluop_hip.grouped_matmul_forward(gpu_handle, xt, w, dev), want[0])
    wv = torch.zeros(4 * 64 * 96 + 1, dtype=torch.bfloat16, device="cuda")[1:].view(4, 64, 96)
    wv.copy_(w)
    a = mluop_hip.grouped_matmul_forward(gpu_handle, x, wv, dev)
    assert torch.allclose(a.float(), want[0].float(), rtol=2.0 ** -7, atol=1e-3)


def test_addresses_beyond_32_bits(gpu_handle):
    """rows and filters that begin more than 4 GiB behind their tensors' first"""
    import torch
    import mluop_hip
    rows, ci, co = (1 << 20) + 300, 2304, 16
    x = torch.zeros(rows, ci, dtype=torch.float16, device="cuda")
    x[-290:] = 1.0
    w = torch.full((2, ci, co), 2.0 ** -10, dtype=torch.float16, device="cuda")
    dev = torch.tensor([0, 1 << 20, rows], dtype=torch.int32, device="cuda")
    y = mluop_hip.grouped_matmul_forward(gpu_handle, x, w, dev)
    assert bool((y[-290:] == 2.25).all()) and not bool(y[:-290].any())
    dx = mluop_hip.grouped_matmul_backward_data(gpu_handle, torch.ones(rows, co, dtype=torch.float16, device="cuda"), w, dev)
    assert bool((dx[-290:] == 2.0 ** -6).all()) and bool((dx[:100] == 2.0 ** -6).all())
    del dx
    dw = mluop_hip.grouped_matmul_backward_filter(gpu_handle, x, torch.ones(rows, co, dtype=torch.float16, device="cuda"), dev)
    assert bool((dw[1] == 290).all()) and not bool(dw[0].any())
    del x, y, dw
    w = torch.zeros(600, 2048, 2048, dtype=torch.float16, device="cuda")
    w[599], w[520] = 2.0 ** -11, 2.0 ** -10
    x = torch.ones(4, 2048, dtype=torch.float16, device="cuda")
    dev = torch.tensor([0] * 521 + [1] * 79 + [4], dtype=torch.int32, device="cuda")
    y = mluop_hip.grouped_matmul_forward(gpu_handle, x, w, dev)
    assert y.mean(dim=1).tolist() == [2.0, 1.0, 1.0, 1.0]
    dx = mluop_hip.grouped_matmul_backward_data(gpu_handle, x, w, dev)
    assert dx.mean(dim=1).tolist() == [2.0, 1.0, 1.0, 1.0]


def test_starts_that_make_no_sense_stay_in_bounds(gpu_handle):
    """(their results are undefined; no access leaves a tensor: outputs lie between guard bands)"""
    import torch
    for rows in (100, 3000):
        x, w, dy = inputs(rows, 4, 64, 64, torch.float16, 5)
        for starts in ([-5, 200, 50, 10, 1000], [100, 50, 20, 10, 0], [0, 1 << 30, -(1 << 30), 7, 7], [0, 3000, 0, 3000, 0]):
            products(gpu_handle, x, w, dy, torch.tensor(starts, dtype=torch.int32, device="cuda"))
    torch.cuda.synchronize()


def test_layer_and_autograd():
    import torch
    from mluop_hip import nn as spnn
    torch.manual_seed(4)
    layer = spnn.ExpertLinear(3, 24, 40).cuda()
    x = torch.randn(90, 24, device="cuda", requires_grad=True)
    starts = torch.tensor([0, 20, 20, 90], dtype=torch.int32, device="cuda")
    y = layer(x, starts)
    ref = torch.cat([x[:20] @ layer.weight[0], x[20:] @ layer.weight[2]])
    assert torch.allclose(y, ref, atol=1e-4)
    dy = torch.randn_like(y)
    for a, b in zip(torch.autograd.grad(y, [x, layer.weight], dy), torch.autograd.grad(ref, [x, layer.weight], dy)):
        assert torch.allclose(a, b, atol=1e-3)
    # along a direction the product is linear: differences are its gradient but for roundings
    d = torch.randn_like(layer.weight)
    values = [float((spnn.grouped_matmul(x.detach(), layer.weight.detach() + s * d, starts).double() * dy.double()).sum())
              for s in (1.0, -1.0)]
    grad = torch.autograd.grad(layer(x, starts), layer.weight, dy)[0]
    assert abs((values[0] - values[1]) / 2 - float((grad.double() * d.double()).sum())) <= 1e-2


def test_captured_and_on_another_stream():
    import torch
    from mluop_hip import nn as spnn
    x = torch.randn(900, 128, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    w = torch.randn(4, 128, 256, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    dy = torch.randn(900, 256, device="cuda", dtype=torch.bfloat16)
    starts = torch.tensor([0, 100, 300, 300, 900], dtype=torch.int32, device="cuda")
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())

    def step():
        y = spnn.grouped_matmul(x, w, starts)
        return (y,) + torch.autograd.grad(y, [x, w], dy)
    with torch.cuda.stream(stream):
        step()
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            got = step()
    torch.cuda.synchronize()
    for k in range(3):
        with torch.no_grad():
            x.copy_(torch.randn_like(x))
        starts[1] = 50 * k
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, step()))


def test_no_rows(gpu_handle):
    import torch
    x, w, dy = inputs(0, 3, 16, 32, torch.float16, 1)
    y, dx, dw = products(gpu_handle, x, w, dy, torch.zeros(4, dtype=torch.int32, device="cuda"))
    assert y.shape == (0, 32) and dx.shape == (0, 16) and not bool(dw.any())


def test_refusals(gpu_handle):
    import torch
    import mluop_hip
    x, w, dy = inputs(10, 2, 16, 32, torch.float16, 1)
    s = torch.tensor([0, 5, 10], dtype=torch.int32, device="cuda")
    f = mluop_hip.grouped_matmul_forward
    for args in ((x.double(), w, s), (x, w.float(), s), (x[:, :8], w, s), (x, w[0], s), (x, w, s[:2]), (x, w, s.long()),
                 (x, w, s.cpu()), (x.cpu(), w, s), (x, w.cpu(), s)):
        with pytest.raises(ValueError):
            f(gpu_handle, *args)
    with pytest.raises(ValueError):
        mluop_hip.grouped_matmul_backward_data(gpu_handle, x, w, s)
    for args in ((x, dy[:5], s), (x, dy.float(), s)):
        with pytest.raises(ValueError):
            mluop_hip.grouped_matmul_backward_filter(gpu_handle, *args)
