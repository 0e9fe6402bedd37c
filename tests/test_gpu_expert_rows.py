"""Rows into the order of their experts and back: the order against a stable sort at every way that sizes take, choices of no expert,
dispatch exactly, weighted sums and gradients against float64, strides, streams, captured graphs; refusals."""
import pytest

pytestmark = pytest.mark.gpu

LAST = {"float32": 2.0 ** -24, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}
LEAST = 2.0 ** -25


def order(chosen, experts):
    """(rows, starts, places) on the host"""
    import numpy as np
    flat = chosen.cpu().numpy().reshape(-1).astype(np.int64)
    flat = np.where((flat >= 0) & (flat < experts), flat, experts)
    by = np.argsort(flat, kind="stable")
    starts = np.searchsorted(flat[by], np.arange(experts + 1))
    places = np.empty_like(by)
    places[by] = np.arange(by.size)
    return np.where(flat[by] < experts, by // chosen.shape[1], -1), starts, np.where(flat < experts, places, -1).reshape(chosen.shape)


@pytest.mark.parametrize("index", ["int32", "int64"])
@pytest.mark.parametrize("rows,choices,experts", [
    (1, 1, 1), (1, 2, 5), (3, 4, 2047), (700, 2, 8), (2048, 1, 64), (2049, 1, 33), (5000, 3, 27), (9000, 8, 512),
    (40_000, 2, 2047), (33_000, 1, 1000), (2_200_000, 1, 16), (300_000, 7, 100)])
def test_order(gpu_handle, index, rows, choices, experts):
    import numpy as np
    import torch
    import mluop_hip
    print("expert order", index, rows, choices, experts, flush=True)
    g = torch.Generator(device="cuda").manual_seed(rows + experts)
    # (uneven, one choice in ten of no expert, and one expert that most rows may name)
    chosen = (experts * torch.rand((rows, choices), device="cuda", generator=g) ** 2).long()
    u = torch.rand((rows, choices), device="cuda", generator=g)
    chosen[u < 0.05] = -1
    chosen[(u >= 0.05) & (u < 0.1)] = experts
    chosen[(u >= 0.1) & (u < 0.12)] = (1 << 40) if index == "int64" else -(1 << 31)
    if rows == 5000:
        chosen[:] = 3
    chosen = chosen.to(getattr(torch, index))
    got = mluop_hip.expert_order(gpu_handle, chosen, experts)
    for a, b in zip(got, order(chosen, experts)):
        assert a.dtype == torch.int32 and np.array_equal(a.cpu().numpy(), b)


def test_order_beside_the_one_without_the_library():
    import torch
    from mluop_hip import nn as spnn
    chosen = torch.randint(-2, 9, (600, 3), device="cuda")
    want = spnn.expert_order(chosen, 7)
    for other in (chosen.cpu(), chosen.to(torch.int16)):
        for a, b in zip(spnn.expert_order(other, 7), want):
            assert a.dtype == b.dtype and torch.equal(a.cpu(), b.cpu())
    assert all(torch.equal(a, b) for a, b in zip(spnn.expert_order(chosen.int(), 7), want))
    many = spnn.expert_order(chosen, 5000)   # (more than the library orders)
    assert many[1].shape == (5001,) and many[1][-1] == int((chosen >= 0).sum())


def routing(rows, choices, experts, seed, dropped=0.1):
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)
    chosen = torch.randint(0, experts, (rows, choices), device="cuda", generator=g, dtype=torch.int32)
    chosen[torch.rand((rows, choices), device="cuda", generator=g) < dropped] = -1
    return chosen, g


def taken(rows, places):
    import torch
    found = rows[places.long().clamp(min=0)].double()
    return torch.where((places >= 0).unsqueeze(-1), found, 0.0)


CASES = [(1, 1, 1, 1), (1, 3, 4, 8), (7, 2, 3, 33), (500, 2, 8, 64), (333, 5, 16, 100), (64, 4, 8, 250), (40, 2, 4, 1024),
         (30, 1, 3, 2056), (3, 9, 10, 4100), (2000, 3, 5, 24)]


@pytest.mark.parametrize("dtype,weight", [("float32", "float32"), ("float16", "float16"), ("bfloat16", "float32"),
                                          ("bfloat16", None)])
@pytest.mark.parametrize("rows,choices,experts,channels", CASES)
def test_rows_and_back(gpu_handle, dtype, weight, rows, choices, experts, channels):
    import torch
    import mluop_hip
    print("expert rows", dtype, weight, rows, choices, experts, channels, flush=True)
    chosen, g = routing(rows, choices, experts, rows + channels)
    kind = getattr(torch, dtype)

    def randn(*shape):
        return torch.randn(*shape, device="cuda", generator=g).to(kind)
    x, y, dy = randn(rows, channels), randn(rows * choices, channels), randn(rows, channels)
    w = None if weight is None else torch.rand(rows, choices, device="cuda", generator=g).to(getattr(torch, weight))
    named, starts, places = mluop_hip.expert_order(gpu_handle, chosen, experts)
    ordered = mluop_hip.expert_dispatch(gpu_handle, x, places, starts)
    assert torch.equal(ordered, mluop_hip.embedding_forward(gpu_handle, x, named))

    def near(got, want, size, units, last):
        room = LAST[last] * want.abs() + units * 2.0 ** -24 * size + LEAST
        off = (got.double() - want).abs()
        assert got.dtype == getattr(torch, last) and bool((off <= room).all()), float((off / room).max())
    of_choice = torch.ones(rows, choices, 1, device="cuda", dtype=torch.float64) if w is None else w.double().unsqueeze(2)
    terms = taken(y, places) * of_choice
    near(mluop_hip.expert_combine(gpu_handle, y, places, w), terms.sum(dim=1), terms.abs().sum(dim=1), choices + 1, dtype)
    terms = taken(y, places)
    near(mluop_hip.expert_combine(gpu_handle, y, places), terms.sum(dim=1), terms.abs().sum(dim=1), choices + 1, dtype)
    dr, dw = mluop_hip.expert_combine_backward(gpu_handle, dy, y, places, w, starts)
    want = torch.zeros(rows * choices, channels, device="cuda", dtype=torch.float64)
    there = places >= 0
    want[places[there].long()] = (dy.double().unsqueeze(1) * of_choice)[there]
    near(dr, want, want.abs(), 1, dtype)
    assert (dw is None) == (w is None)
    if w is not None:
        terms = dy.double().unsqueeze(1) * taken(y, places)
        near(dw, terms.sum(dim=2), terms.abs().sum(dim=2), channels + 8, weight)


def test_autograd():
    import torch
    from mluop_hip import nn as spnn
    chosen, g = routing(200, 3, 6, 1)
    _, starts, places = spnn.expert_order(chosen, 6)

    def randn(*shape):
        return torch.randn(*shape, device="cuda", generator=g)
    x, w, weight = randn(200, 40).requires_grad_(), randn(200, 3).requires_grad_(), randn(40)
    out = spnn.expert_combine(torch.tanh(spnn.expert_dispatch(x, places, starts)) * weight, places, starts, w)
    x2, w2 = x.detach().double().requires_grad_(), w.detach().double().requires_grad_()
    there = (places >= 0).double().unsqueeze(2)
    want = (torch.tanh(x2).unsqueeze(1) * weight.double() * w2.unsqueeze(2) * there).sum(dim=1)
    assert torch.allclose(out.double(), want, atol=1e-5)
    dy = randn(200, 40)
    for a, b in zip(torch.autograd.grad(out, [x, w], dy), torch.autograd.grad(want, [x2, w2], dy.double())):
        assert torch.allclose(a.double(), b, atol=2e-5)
    # the weights alone, and the results alone
    results = torch.tanh(x.detach()).repeat(3, 1)
    for leaf in (w.detach().clone().requires_grad_(), results.clone().requires_grad_()):
        of = (results, leaf) if leaf.shape == w.shape else (leaf, w.detach())
        (grad,) = torch.autograd.grad(spnn.expert_combine(of[0], places, starts, of[1]), leaf, dy)
        assert grad.shape == leaf.shape and bool(torch.isfinite(grad).all())


def test_a_choice_without_a_place_does_not_count(gpu_handle):
    import torch
    import mluop_hip
    chosen = torch.tensor([[0, -1], [-1, -1], [1, 0]], dtype=torch.int32, device="cuda")
    named, starts, places = mluop_hip.expert_order(gpu_handle, chosen, 2)
    assert named.tolist() == [0, 2, 2, -1, -1, -1] and starts.tolist() == [0, 2, 3]
    assert places.tolist() == [[0, -1], [-1, -1], [2, 1]]
    y = torch.full((6, 8), float("nan"), device="cuda")
    y[:3] = torch.arange(3.0, device="cuda").unsqueeze(1)
    w = torch.full((3, 2), float("inf"), device="cuda")
    w[0, 0], w[2] = 2.0, torch.tensor([3.0, 4.0], device="cuda")
    out = mluop_hip.expert_combine(gpu_handle, y, places, w)
    assert out[:, 0].tolist() == [0.0, 0.0, 10.0]
    dr, dw = mluop_hip.expert_combine_backward(gpu_handle, torch.ones(3, 8, device="cuda"), y, places, w, starts)
    assert dr[:, 0].tolist() == [2.0, 4.0, 3.0, 0.0, 0.0, 0.0] and dw.tolist() == [[0.0, 0.0], [0.0, 0.0], [16.0, 8.0]]


def test_places_that_make_no_sense_stay_in_bounds(gpu_handle):
    """(their results are undefined; no access leaves a tensor: outputs lie between guard bands)"""
    import torch
    import mluop_hip
    x, y = torch.randn(100, 24, device="cuda"), torch.randn(200, 24, device="cuda")
    w = torch.rand(100, 2, device="cuda")
    for fill in (-5, 0, 199, 200, 2 ** 31 - 1, -2 ** 31):
        places = torch.full((100, 2), fill, dtype=torch.int32, device="cuda")
        for end in (-9, 0, 200, 1 << 30):
            starts = torch.tensor([0, end], dtype=torch.int32, device="cuda")
            mluop_hip.expert_dispatch(gpu_handle, x, places, starts)
            mluop_hip.expert_combine_backward(gpu_handle, x, y, places, w, starts)
        mluop_hip.expert_combine(gpu_handle, y, places, w)
    torch.cuda.synchronize()


def test_rows_apart_and_unaligned(gpu_handle):
    import torch
    import mluop_hip
    chosen, g = routing(150, 2, 4, 3)
    _, starts, places = mluop_hip.expert_order(gpu_handle, chosen, 4)

    def randn(*shape):
        return torch.randn(*shape, device="cuda", generator=g).half()
    x, y, w = randn(150, 64), randn(300, 64), torch.rand(150, 2, device="cuda", generator=g)
    want = (mluop_hip.expert_dispatch(gpu_handle, x, places, starts), mluop_hip.expert_combine(gpu_handle, y, places, w),
            *mluop_hip.expert_combine_backward(gpu_handle, x, y, places, w, starts))

    def views(t):
        n = t.shape[0]
        flat = torch.zeros(n * 64 + 1, dtype=t.dtype, device="cuda")
        wide = torch.zeros(2 * n, 160, dtype=t.dtype, device="cuda")
        for view in (wide[::2, 16:80], wide[::2, 3:67], flat[1:].view(n, 64)):
            yield view.copy_(t)
    for a, b in zip(views(x), views(y)):
        got = (mluop_hip.expert_dispatch(gpu_handle, a, places, starts), mluop_hip.expert_combine(gpu_handle, b, places, w),
               *mluop_hip.expert_combine_backward(gpu_handle, a, b, places, w, starts))
        assert all(torch.allclose(c.float(), d.float(), rtol=2.0 ** -10, atol=2.0 ** -14) for c, d in zip(got, want))
    # a mask of choices that lies column by column
    assert torch.equal(mluop_hip.expert_order(gpu_handle, chosen.t().contiguous().t(), 4)[2], places)


def test_no_rows(gpu_handle):
    import torch
    import mluop_hip
    none = torch.zeros(0, 2, dtype=torch.int32, device="cuda")
    named, starts, places = mluop_hip.expert_order(gpu_handle, none, 3)
    assert named.shape == (0,) and places.shape == (0, 2) and starts.tolist() == [0, 0, 0, 0]
    x = torch.zeros(0, 16, device="cuda")
    assert mluop_hip.expert_dispatch(gpu_handle, x, places, starts).shape == (0, 16)
    assert mluop_hip.expert_combine(gpu_handle, x, places).shape == (0, 16)
    dr, dw = mluop_hip.expert_combine_backward(gpu_handle, x, x, places, none.float(), starts)
    assert dr.shape == (0, 16) and dw.shape == (0, 2)


@pytest.mark.parametrize("rows", [50, 9000])
def test_expert_layer_captured(rows):
    """routing, both layers and all gradients in one graph"""
    import torch
    from mluop_hip import nn as spnn
    torch.manual_seed(0)
    layer = spnn.ExpertMLP(32, 48, experts=6, choices=2).cuda()
    x, dy = (torch.randn(rows, 32, device="cuda").bfloat16() for _ in range(2))
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())

    def step():
        leaf = x.detach().requires_grad_()
        out = layer(leaf)
        return [out] + list(torch.autograd.grad(out, [leaf, layer.gate.weight, layer.up.weight], dy))
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
        for a, b in zip(out, step()):
            # (the library product of the gate may take another way inside a graph)
            assert torch.allclose(a.float(), b.float(), rtol=2.0 ** -6, atol=2.0 ** -6 * float(b.float().abs().max()))


def test_refusals(gpu_handle):
    import torch
    import mluop_hip
    chosen, g = routing(20, 2, 4, 3)
    named, starts, places = mluop_hip.expert_order(gpu_handle, chosen, 4)
    x, y, w = torch.randn(20, 8, device="cuda"), torch.randn(40, 8, device="cuda"), torch.rand(20, 2, device="cuda")
    for bad in (chosen.float(), chosen.short(), chosen[0], chosen[:, :0], chosen.cpu()):
        with pytest.raises(ValueError):
            mluop_hip.expert_order(gpu_handle, bad, 4)
    for experts in (0, -1, 2048):
        with pytest.raises(mluop_hip.MluOpError):
            mluop_hip.expert_order(gpu_handle, chosen, experts)
    for bad in (dict(features=x.double()), dict(features=x[:5]), dict(features=x[0]), dict(places=places.long()),
                dict(places=places[0]), dict(group_starts=starts.long()), dict(group_starts=starts[:1]), dict(places=places.cpu())):
        with pytest.raises(ValueError):
            mluop_hip.expert_dispatch(gpu_handle, **{**dict(features=x, places=places, group_starts=starts), **bad})
    for bad in (dict(results=y[:20]), dict(results=y.double()), dict(weights=w[:, :1]), dict(weights=w.half()),
                dict(weights=w.cpu())):
        with pytest.raises(ValueError):
            mluop_hip.expert_combine(gpu_handle, **{**dict(results=y, places=places, weights=w), **bad})
    for bad in (dict(output_grad=x.half()), dict(output_grad=y), dict(results=x)):
        with pytest.raises(ValueError):
            mluop_hip.expert_combine_backward(gpu_handle, **{**dict(output_grad=x, results=y, places=places, weights=w,
                                                                    group_starts=starts), **bad})
