"""The gated recurrence: states and gradients against a float64 recurrence row by row, samples of no rows, of one and across many
tiles, rows of no sample, both directions and kinds, gates at the ends of their range, values that are not finite; single steps;
strides, streams, captured graphs; refusals."""
import pytest

pytestmark = pytest.mark.gpu

LAST = {"float32": 2.0 ** -24, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}
LEAST = {"float32": 2.0 ** -126, "float16": 2.0 ** -25, "bfloat16": 2.0 ** -126}


def inputs(rows, channels, samples, dtype, kind, seed, spread=1.5):
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)

    def randn(*shape):
        return torch.randn(*shape, device="cuda", generator=g)
    gates = 1.5 + spread * randn(rows, channels) if kind == "sigmoid" else -torch.exp(spread * randn(rows, channels) - 2.0)
    return (randn(rows, channels).to(dtype), gates.to(dtype), randn(samples, channels), randn(rows, channels).to(dtype),
            randn(samples, channels))


def host(t):
    return None if t is None else t.detach().double().cpu().numpy()


def within(name, got, want, dtype):
    import torch
    value, room = (torch.from_numpy(v).to(got.device) for v in want)
    dtype = "float32" if got.dtype == torch.float32 else dtype
    room = room + LAST[dtype] * (value.abs() + room) + LEAST[dtype]
    off = (got.double() - value).abs()
    assert bool((off <= room).all()), (name, float((off / room).max()))


def check(handle, x, g, starts, h0, dh, df, kind, reverse, dtype):
    import torch
    import mluop_hip
    from scan_reference import scan
    dev = None if starts is None else torch.tensor(starts, dtype=torch.int32, device="cuda")
    out, final, carries = mluop_hip.gated_scan_forward(handle, x, g, dev, h0, kind, reverse)
    grads = mluop_hip.gated_scan_backward(handle, dh, df, x, g, carries, dev, kind, reverse)
    want = scan(host(x), host(g), starts or [0, x.shape[0]], host(h0), kind, reverse, host(dh), host(df))
    for name, got in zip(("out", "final", "features_grad", "gates_grad", "initial_grad"), (out, final) + tuple(grads)):
        within(name, got, want[name], dtype)
    return out, final, grads


CASES = [  # rows, channels, starts
    (1, 1, None), (1, 64, None), (2, 8, None), (255, 16, None), (256, 64, None), (257, 64, None), (300, 33, None),
    (64, 40, list(range(65))), (513, 7, [0, 0, 1, 256, 513, 513]), (900, 72, [5, 300, 300, 870]), (3001, 64, None),
    (1024, 100, [0, 256, 512, 513, 1024]), (700, 250, [0, 700]), (40, 1000, [0, 17, 40]), (9000, 24, [0, 4500, 9000]),
    (500, 20, [500, 500]), (600, 16, [0] + list(range(0, 600, 2)) + [600])]


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("kind", ["sigmoid", "exp"])
@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("rows,channels,starts", CASES)
def test_against_float64(gpu_handle, dtype, kind, reverse, rows, channels, starts):
    import torch
    samples = 1 if starts is None else len(starts) - 1
    print("gated scan", dtype, kind, reverse, rows, channels, samples, flush=True)
    x, g, h0, dh, df = inputs(rows, channels, samples, getattr(torch, dtype), kind, rows + channels)
    states = (rows + channels) % 3 != 0
    check(gpu_handle, x, g, starts, h0 if states else None, dh, df if states else None, kind, reverse, dtype)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("rows", [40_000, 70_001])
def test_long_memories(gpu_handle, dtype, rows):
    """decays of 1 - 2^-12 and nearer to one, over hundreds of tiles"""
    import torch
    x, g, h0, dh, df = inputs(rows, 8, 1, getattr(torch, dtype), "sigmoid", 3)
    g = (8.0 + 3.0 * torch.rand_like(g.float())).to(g.dtype)
    check(gpu_handle, x, g, None, h0, dh, df, "sigmoid", False, dtype)


@pytest.mark.parametrize("kind", ["sigmoid", "exp"])
@pytest.mark.parametrize("reverse", [False, True])
def test_gates_at_the_ends_of_their_range(gpu_handle, kind, reverse):
    """a decay of exactly zero cuts a sample, one of exactly one keeps it"""
    import torch
    x, g, h0, dh, df = inputs(700, 16, 1, torch.float32, kind, 11)
    g[::50, 3] = float("-inf")
    g[::50, 4] = -200.0
    g[:, 5] = float("inf") if kind == "sigmoid" else 0.0
    g[:, 6] = 100.0 if kind == "sigmoid" else -1e-30
    import numpy as np
    with np.errstate(over="ignore"):
        out, final, grads = check(gpu_handle, x, g, None, h0, dh, df, kind, reverse, "float32")
    assert all(bool(torch.isfinite(t).all()) for t in (out, final) + tuple(grads))
    if kind == "sigmoid":   # nothing but the initial state is left in it
        assert torch.equal(out[:, 5], h0[0, 5].expand(700)) and not bool(grads[0][:, 5].any())


@pytest.mark.parametrize("reverse", [False, True])
def test_values_that_are_not_finite_stay_behind_their_row(gpu_handle, reverse):
    import torch
    import mluop_hip
    x, g, h0, dh, df = inputs(1500, 16, 2, torch.float32, "sigmoid", 4)
    starts = torch.tensor([0, 900, 1500], dtype=torch.int32, device="cuda")
    args = (starts, h0, "sigmoid", reverse)
    out, final, carries = mluop_hip.gated_scan_forward(gpu_handle, x, g, *args)
    grads = mluop_hip.gated_scan_backward(gpu_handle, dh, df, x, g, carries, starts, "sigmoid", reverse)
    x2, dh2 = x.clone(), dh.clone()
    x2[400, 3], dh2[500, 5] = float("nan"), float("inf")
    out2, final2, carries2 = mluop_hip.gated_scan_forward(gpu_handle, x2, g, *args)
    grads2 = mluop_hip.gated_scan_backward(gpu_handle, dh2, df, x2, g, carries2, starts, "sigmoid", reverse)
    rows = torch.arange(1500, device="cuda")
    behind = (rows <= 400) if reverse else (rows >= 400) & (rows < 900)
    other = torch.ones(16, dtype=torch.bool, device="cuda")
    other[3] = False
    assert torch.equal(out2[:, other], out[:, other]) and torch.equal(out2[~behind], out[~behind])
    assert bool(torch.isnan(out2[behind, 3]).all()) and torch.equal(final2[1], final[1])
    # the gradient comes the other way
    through = (rows >= 500) & (rows < 900) if reverse else rows <= 500
    other[5] = False
    assert torch.equal(grads2[0][~through], grads[0][~through]) and torch.equal(grads2[0][:, other], grads[0][:, other])
    assert not bool(torch.isfinite(grads2[0][through, 5]).any()) and torch.equal(grads2[2][1], grads[2][1])


def test_rows_of_no_sample_are_not_read_and_zero(gpu_handle):
    import torch
    import mluop_hip
    x, g, h0, dh, df = inputs(1000, 24, 3, torch.float16, "exp", 6)
    starts = torch.tensor([100, 400, 400, 930], dtype=torch.int32, device="cuda")
    for t in (x, g, dh):
        t[:100], t[930:] = float("nan"), float("inf")
    out, final, carries = mluop_hip.gated_scan_forward(gpu_handle, x, g, starts, h0, "exp")
    grads = mluop_hip.gated_scan_backward(gpu_handle, dh, df, x, g, carries, starts, "exp")
    for t in (out, grads[0], grads[1]):
        assert not bool(t[:100].any()) and not bool(t[930:].any()) and bool(torch.isfinite(t).all())
    assert torch.equal(final[1], h0[1]) and torch.equal(grads[2][1], df[1])


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("reverse", [False, True])
def test_step_by_step(gpu_handle, dtype, reverse):
    """sequences taken a row at a time, with the states handed on, end as they do in one call"""
    import torch
    import mluop_hip
    x, g, h0, _, _ = inputs(5 * 12, 48, 5, getattr(torch, dtype), "sigmoid", 7)
    starts = torch.arange(0, 61, 12, dtype=torch.int32, device="cuda")
    out, final, _ = mluop_hip.gated_scan_forward(gpu_handle, x, g, starts, h0, "sigmoid", reverse)
    state, ones = h0, torch.arange(6, dtype=torch.int32, device="cuda")
    order = range(11, -1, -1) if reverse else range(12)
    for t in order:
        y, state, _ = mluop_hip.gated_scan_forward(gpu_handle, x[t::12], g[t::12], ones, state, "sigmoid")
        assert torch.allclose(y.float(), out[t::12].float(), rtol=2.0 ** -7 if dtype == "bfloat16" else 2.0 ** -19, atol=2.0 ** -18)
    assert torch.allclose(state, final, rtol=2.0 ** -19, atol=2.0 ** -19)


def test_gradient_by_differences(gpu_handle):
    import numpy as np
    import torch
    import mluop_hip
    from scan_reference import scan
    for kind in ("sigmoid", "exp"):
        x, g, h0, dh, df = inputs(300, 6, 2, torch.float32, kind, 9)
        starts = [0, 270, 300]
        dev = torch.tensor(starts, dtype=torch.int32, device="cuda")
        carries = mluop_hip.gated_scan_forward(gpu_handle, x, g, dev, h0, kind)[2]
        grads = mluop_hip.gated_scan_backward(gpu_handle, dh, df, x, g, carries, dev, kind)
        rng = np.random.default_rng(0)
        for k in range(3):
            args = [host(x), host(g), host(h0)]
            d, h, values = rng.standard_normal(args[k].shape), 2.0 ** -10, []
            for s in (1, -1):
                moved = [v + s * h * d if i == k else v for i, v in enumerate(args)]
                got = scan(moved[0], moved[1], starts, moved[2], kind, False)
                values.append(float((got["out"][0] * host(dh)).sum() + (got["final"][0] * host(df)).sum()))
            slope, want = (values[0] - values[1]) / (2 * h), float((host(grads[k]) * d).sum())
            assert abs(slope - want) <= 1e-3 * (abs(want) + np.linalg.norm(d))


def test_autograd_and_missing_gradients():
    import torch
    from mluop_hip import nn as spnn
    x, g, h0, dh, df = inputs(400, 16, 1, torch.float32, "sigmoid", 12)
    leaves = [t.clone().requires_grad_() for t in (x, g, h0)]
    out, final = spnn.gated_scan(leaves[0], leaves[1], None, leaves[2])
    both = torch.autograd.grad([out, final], leaves, [dh, df], retain_graph=True)
    of_out = torch.autograd.grad(out, leaves, dh, retain_graph=True)
    of_final = torch.autograd.grad(final, leaves, df)
    for a, b, c in zip(both, of_out, of_final):
        assert torch.allclose(a, b + c, rtol=1e-4, atol=1e-5)
    # a view of every second column block, as a projection's two halves are
    wide = torch.randn(400, 32, device="cuda", requires_grad=True)
    a, b = wide.chunk(2, dim=1)
    out = spnn.gated_scan(a, b, kind="sigmoid", reverse=True)[0]
    assert torch.equal(out, spnn.gated_scan(a.contiguous(), b.contiguous(), reverse=True)[0])
    out.sum().backward()
    assert bool(torch.isfinite(wide.grad).all())


def test_rows_apart_and_unaligned(gpu_handle):
    import torch
    import mluop_hip
    x, g, h0, dh, df = inputs(700, 64, 1, torch.float16, "sigmoid", 13)
    want = mluop_hip.gated_scan_forward(gpu_handle, x, g, None, h0)
    grads = mluop_hip.gated_scan_backward(gpu_handle, dh, df, x, g, want[2])
    wide = torch.zeros(1400, 160, dtype=torch.float16, device="cuda")
    flat = torch.zeros(700 * 64 + 1, dtype=torch.float16, device="cuda")
    for view in (wide[::2, 16:80], wide[::2, 3:67], flat[1:].view(700, 64)):
        view.copy_(x)
        got = mluop_hip.gated_scan_forward(gpu_handle, view, g, None, h0)
        # (other vectors, other compositions; the carries of one alignment serve the other)
        again = mluop_hip.gated_scan_backward(gpu_handle, dh, df, view, g, want[2])
        for a, c in zip(got[:2] + again, want[:2] + grads):
            assert torch.allclose(a.float(), c.float(), rtol=2.0 ** -10, atol=2.0 ** -14)
    one = g[:1].expand(700, 64)
    assert torch.equal(mluop_hip.gated_scan_forward(gpu_handle, x, one)[0],
                       mluop_hip.gated_scan_forward(gpu_handle, x, one.contiguous())[0])


def test_starts_that_make_no_sense_stay_in_bounds(gpu_handle):
    """(their results are undefined; no access leaves a tensor: outputs lie between guard bands)"""
    import torch
    import mluop_hip
    x, g, h0, dh, df = inputs(3000, 16, 5, torch.float16, "sigmoid", 2)
    for starts in ([0, 3000, 0, 3000, 0, 3000], [-7, 1 << 30, 5, 4, 3, 2], [9] * 6, [3000, 0, -1, 3000, 0, 1]):
        dev = torch.tensor(starts, dtype=torch.int32, device="cuda")
        for reverse in (False, True):
            out, final, carries = mluop_hip.gated_scan_forward(gpu_handle, x, g, dev, h0, "sigmoid", reverse)
            mluop_hip.gated_scan_backward(gpu_handle, dh, df, x, g, carries, dev, "sigmoid", reverse)
    torch.cuda.synchronize()


def test_no_rows(gpu_handle):
    import torch
    import mluop_hip
    x, h0 = torch.zeros(0, 40, device="cuda"), torch.randn(3, 40, device="cuda")
    starts = torch.zeros(4, dtype=torch.int32, device="cuda")
    out, final, carries = mluop_hip.gated_scan_forward(gpu_handle, x, x, starts, h0)
    assert out.shape == (0, 40) and torch.equal(final, h0)
    dx, dg, di = mluop_hip.gated_scan_backward(gpu_handle, x, h0, x, x, carries, starts)
    assert dx.shape == dg.shape == (0, 40) and torch.equal(di, h0)
    assert not bool(mluop_hip.gated_scan_forward(gpu_handle, x, x)[1].any())


@pytest.mark.parametrize("rows", [200, 5000])
def test_captured_with_its_gradients(rows):
    import torch
    from mluop_hip import nn as spnn
    x, g, h0, dh, df = inputs(rows, 64, 2, torch.float16, "sigmoid", 3)
    starts = torch.tensor([0, rows // 3, rows], dtype=torch.int32, device="cuda")
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())

    def step():
        leaves = [t.detach().requires_grad_() for t in (x, g, h0)]
        y = spnn.gated_scan(leaves[0], leaves[1], starts, leaves[2])
        return list(y) + list(torch.autograd.grad(y, leaves, [dh, df]))
    with torch.cuda.stream(stream):
        step()
        stream.synchronize()
        graphs = []
        for _ in range(2):
            graphs.append(torch.cuda.CUDAGraph())
            with torch.cuda.graph(graphs[-1], stream=stream):
                out = step()
            graphs[-1].out = out
    torch.cuda.synchronize()
    for k in range(4):
        x.copy_(torch.randn_like(x))
        starts[1] = 100 + k
        graphs[0].replay()
        graphs[1].replay()
        torch.cuda.synchronize()
        want = step()
        for graph in graphs:
            assert all(torch.equal(a, c) for a, c in zip(graph.out, want))


def test_module():
    import torch
    from mluop_hip import nn as spnn
    torch.manual_seed(2)
    for kind in ("sigmoid", "exp"):
        layer = spnn.GatedScan(16, 24, kind).cuda()
        rows = torch.randn(90, 16, device="cuda", requires_grad=True)
        starts = torch.tensor([0, 40, 90], dtype=torch.int32, device="cuda")
        out, final = layer(rows, starts, states=True)
        # in two pieces, the second from the first's states
        cut = torch.tensor([0, 30, 65], dtype=torch.int32, device="cuda")
        at = torch.cat([torch.arange(0, 30), torch.arange(40, 75)]).cuda()
        rest = torch.cat([torch.arange(30, 40), torch.arange(75, 90)]).cuda()
        first, states = layer(rows[at], cut, states=True)
        second, last = layer(rows[rest], torch.tensor([0, 10, 25], dtype=torch.int32, device="cuda"), states, states=True)
        assert torch.allclose(first, out[at], atol=1e-5) and torch.allclose(second, out[rest], atol=1e-5)
        assert torch.allclose(last, final, atol=1e-5)
        out.square().sum().backward()
        assert all(bool(torch.isfinite(p.grad).all()) for p in layer.parameters())
    # a SparseTensor whose rows are in no order gives what it gives in order
    idx = torch.tensor([[n, 0, i // 5, i % 5] for n in range(2) for i in range(20)], dtype=torch.int32, device="cuda")
    feats, mixed = torch.randn(40, 16, device="cuda"), torch.randperm(40, device="cuda")
    net = spnn.SparseSequential(spnn.GatedScan(16, kind="exp", reverse=True).cuda())
    want = net[0](feats, torch.tensor([0, 20, 40], dtype=torch.int32, device="cuda"))
    got = net(spnn.SparseTensor(feats, idx, (1, 5, 5), 2, distinct=True)).features
    assert torch.allclose(got, want, atol=1e-6)
    # (the order within a sample is that of its rows)
    sample = torch.cat([mixed[mixed < 20], mixed[mixed >= 20]])
    got = net(spnn.SparseTensor(feats[mixed], idx[mixed], (1, 5, 5), 2, distinct=True)).features
    again = net[0](feats[sample], torch.tensor([0, 20, 40], dtype=torch.int32, device="cuda"))
    places = torch.empty(40, dtype=torch.long, device="cuda")
    places[sample] = torch.arange(40, device="cuda")
    assert torch.allclose(got, again[places[mixed]], atol=1e-6)


def test_refusals(gpu_handle):
    import torch
    import mluop_hip
    x, g, h0, dh, df = inputs(10, 8, 1, torch.float16, "sigmoid", 1)
    f = mluop_hip.gated_scan_forward
    starts = torch.tensor([0, 10], dtype=torch.int32, device="cuda")
    for bad in (dict(features=x.double()), dict(features=x[0]), dict(features=x.cpu()), dict(gates=g[:5]), dict(gates=g.float()),
                dict(row_starts=starts.long()), dict(row_starts=starts[:1]), dict(row_starts=starts.cpu()),
                dict(initial=h0.half()), dict(initial=h0[:, :4]), dict(initial=h0[0])):
        with pytest.raises(ValueError):
            f(gpu_handle, **{**dict(features=x, gates=g, row_starts=starts, initial=h0), **bad})
    with pytest.raises(KeyError):
        f(gpu_handle, x, g, kind="tanh")
    carries = f(gpu_handle, x, g)[2]
    for bad in (dict(carries=carries[:0]), dict(carries=carries.half()), dict(output_grad=dh[:5]), dict(final_grad=df.half()),
                dict(output_grad=dh.float())):
        with pytest.raises(ValueError):
            mluop_hip.gated_scan_backward(gpu_handle, **{**dict(output_grad=dh, final_grad=df, features=x, gates=g,
                                                                carries=carries), **bad})
