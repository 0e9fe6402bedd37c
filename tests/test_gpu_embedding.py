"""Embedding lookup with scaling and the gradient of its table: exact where every result is one product, the gradient
against float64 sums at rows named never, once, around a piece and by every token; tokens that name no row, strides, both
token types, addresses beyond 32 bits, and the layer with autograd."""
import pytest

pytestmark = pytest.mark.gpu

LAST = {"float32": 2.0 ** -24, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}


def reference_grad(grad, tokens, rows, scale):
    import torch
    named = (tokens >= 0) & (tokens < rows)
    out = torch.zeros(rows, grad.shape[1], dtype=torch.float64)
    sizes = torch.zeros_like(out)
    g = grad.double().cpu()[named.cpu()]
    at = tokens[named].long().cpu()
    return out.index_add_(0, at, g) * scale, sizes.index_add_(0, at, g.abs()) * abs(scale), torch.bincount(at, minlength=rows)


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("channels", [1, 2, 3, 8, 33, 64, 1024, 2056, 4100])
@pytest.mark.parametrize("tokens,wide", [(1, False), (5, True), (64, False), (1000, True)])
def test_forward(gpu_handle, dtype, channels, tokens, wide):
    import torch
    import mluop_hip
    print("embedding", dtype, channels, tokens, wide, flush=True)
    g = torch.Generator(device="cuda").manual_seed(channels + tokens)
    dtype = getattr(torch, dtype)
    table = torch.randn(77, channels, device="cuda", generator=g).to(dtype)
    t = torch.randint(-3, 80, (tokens,), device="cuda", generator=g, dtype=torch.int64 if wide else torch.int32)
    if wide:
        t[0] = 1 << 40
    got = mluop_hip.embedding_forward(gpu_handle, table, t, 1.7)
    named = (t >= 0) & (t < 77)
    # one product in float32 (of the float32 scale) and one rounding
    want = (table[torch.where(named, t, torch.zeros_like(t)).long()].float() * torch.tensor(1.7, device="cuda")).to(dtype)
    assert torch.equal(got, torch.where(named[:, None], want, torch.zeros_like(want)))


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("channels", [1, 6, 33, 64, 520, 2056])
@pytest.mark.parametrize("rows,tokens", [(1, 1), (1, 1000), (7, 64), (7, 65), (300, 129), (1025, 5000), (70000, 3000),
                                         (40, 20000)])
def test_gradient(gpu_handle, dtype, channels, rows, tokens):
    import torch
    import mluop_hip
    if channels * tokens > 1 << 23:
        tokens = (1 << 23) // channels
    print("embedding grad", dtype, channels, rows, tokens, flush=True)
    g = torch.Generator(device="cuda").manual_seed(rows + tokens)
    # half of them a few rows, a tenth none
    t = torch.randint(0, rows, (tokens,), device="cuda", generator=g, dtype=torch.int32)
    pick = torch.rand(tokens, device="cuda", generator=g)
    t = torch.where(pick < 0.5, t % 3, t)
    t = torch.where(pick > 0.9, torch.where(pick > 0.95, rows, -1).to(torch.int32), t)
    t = t.clamp(max=rows)
    grad = torch.randn(tokens, channels, device="cuda", generator=g).to(getattr(torch, dtype))
    got = mluop_hip.embedding_backward(gpu_handle, grad, t, rows, 0.5)
    want, sizes, counts = reference_grad(grad, t, rows, 0.5)
    # a sum of n terms in any fixed order is off by at most n halves of a unit of the sum of their magnitudes
    room = (counts[:, None] + 1.0) * 2.0 ** -24 * sizes + LAST[dtype] * (want.abs() + 1e-6) + 2.0 ** -25
    assert bool(((got.double().cpu() - want).abs() <= room).all())
    assert bool((got.cpu()[counts == 0] == 0).all())
    assert torch.equal(got, mluop_hip.embedding_backward(gpu_handle, grad, t.long(), rows, 0.5))


@pytest.mark.parametrize("lengths", [[64, 64, 64], [65], [63, 65, 64, 1, 128, 129], [1, 64, 1, 64, 200], [127, 1, 66],
                                     [64 * 40 + 1, 1, 64 * 7 - 1], [32, 96, 32, 96], [1] * 64 + [65] + [1] * 63])
def test_rows_around_pieces(gpu_handle, lengths):
    """every row's run begins and ends at all places of a piece: integers, so that sums are exact"""
    import torch
    import mluop_hip
    g = torch.Generator(device="cuda").manual_seed(len(lengths))
    tokens = torch.cat([torch.full((n,), v, dtype=torch.int32) for v, n in enumerate(lengths)]).cuda()
    perm = torch.randperm(tokens.numel(), generator=g, device="cuda")
    grad = torch.randint(-8, 9, (tokens.numel(), 40), device="cuda", generator=g).float()
    rows = len(lengths) + 3
    want = torch.zeros(rows, 40, device="cuda").index_add_(0, tokens.long(), grad)
    for order in (torch.arange(tokens.numel(), device="cuda"), perm):
        got = mluop_hip.embedding_backward(gpu_handle, grad[order].contiguous(), tokens[order].contiguous(), rows)
        assert torch.equal(got, want)


def test_no_tokens_and_none_that_names_a_row(gpu_handle):
    import torch
    import mluop_hip
    table = torch.randn(5, 8, device="cuda")
    none = torch.zeros(0, dtype=torch.int32, device="cuda")
    assert mluop_hip.embedding_forward(gpu_handle, table, none).shape == (0, 8)
    assert not bool(mluop_hip.embedding_backward(gpu_handle, torch.zeros(0, 8, device="cuda"), none, 5).any())
    t = torch.full((200,), -1, dtype=torch.int32, device="cuda")
    nan = torch.full((200, 8), float("nan"), device="cuda")
    assert not bool(mluop_hip.embedding_forward(gpu_handle, nan[:5], t, float("inf")).any())
    assert not bool(mluop_hip.embedding_backward(gpu_handle, nan, t, 5).any())


def test_values_that_are_not_finite_stay_in_their_rows(gpu_handle):
    import torch
    import mluop_hip
    grad = torch.ones(300, 8, device="cuda")
    t = (torch.arange(300, device="cuda") % 3).to(torch.int32)
    grad[3, 1], grad[4, 2] = float("inf"), float("nan")
    got = mluop_hip.embedding_backward(gpu_handle, grad, t, 4)
    want = torch.full((4, 8), 100.0, device="cuda")
    want[3], want[0, 1], want[1, 2] = 0.0, float("inf"), float("nan")
    assert torch.equal(torch.nan_to_num(got, nan=-1.0), torch.nan_to_num(want, nan=-1.0))


def test_strides_and_alignment(gpu_handle):
    import torch
    import mluop_hip
    wide = torch.randn(50, 80, device="cuda").half()
    t = torch.randint(0, 50, (90,), device="cuda", dtype=torch.int32)
    for view in (wide[:, 8:40], wide[:, 3:35], wide[::2, 16:48], wide.t()[:32].t()):
        rows = view.shape[0]
        tt = t % rows
        assert torch.equal(mluop_hip.embedding_forward(gpu_handle, view, tt, 2.0), view[tt.long()] * 2)
    grad = torch.randn(90, 80, device="cuda").half()
    for view in (grad[:, 8:40], grad[:, 1:33]):
        assert torch.equal(mluop_hip.embedding_backward(gpu_handle, view, t, 50),
                           mluop_hip.embedding_backward(gpu_handle, view.contiguous(), t, 50))


def test_addresses_beyond_32_bits(gpu_handle):
    import torch
    import mluop_hip
    table = torch.zeros((1 << 19) + 3, 4096, dtype=torch.bfloat16, device="cuda")
    table[-1], table[1 << 18] = 3.0, 5.0
    t = torch.tensor([(1 << 19) + 2, 1 << 18, 0], dtype=torch.int32, device="cuda")
    assert mluop_hip.embedding_forward(gpu_handle, table, t)[:, 7].tolist() == [3.0, 5.0, 0.0]
    del table
    grad = torch.ones(3, 4096, dtype=torch.bfloat16, device="cuda")
    got = mluop_hip.embedding_backward(gpu_handle, grad, t, (1 << 19) + 3)
    assert bool((got[-1] == 1).all()) and bool((got[1 << 18] == 1).all()) and bool((got[0] == 1).all())
    assert float(got[:, ::1024].float().sum()) == 12.0


def test_layer_and_autograd():
    import torch
    from mluop_hip import nn as spnn
    torch.manual_seed(2)
    layer = spnn.Embedding(30, 12, scale=2.5).cuda()
    t = torch.randint(0, 30, (4, 25), device="cuda")
    t[0, 0] = -1
    out = layer(t)
    assert out.shape == (4, 25, 12) and not bool(out[0, 0].any())
    dy = torch.randn_like(out)
    (grad,) = torch.autograd.grad(out, layer.weight, dy)
    ref = torch.nn.functional.embedding(t.clamp(min=0), layer.weight) * 2.5 * (t >= 0).unsqueeze(-1)
    (want,) = torch.autograd.grad(ref, layer.weight, dy)
    assert torch.allclose(out, ref, atol=1e-6) and torch.allclose(grad, want, atol=1e-4)
    # and against differences
    d = torch.randn_like(layer.weight)
    h = 2.0 ** -6
    values = [float((spnn.embedding(layer.weight.detach() + s * h * d, t, 2.5).double() * dy.double()).sum()) for s in (1, -1)]
    assert abs((values[0] - values[1]) / (2 * h) - float((grad.double() * d.double()).sum())) <= 1e-3 * float(d.norm()) * 10


def test_captured():
    import torch
    from mluop_hip import nn as spnn
    table = torch.randn(500, 64, device="cuda", requires_grad=True)
    t = torch.randint(0, 500, (700,), device="cuda", dtype=torch.int32)
    dy = torch.randn(700, 64, device="cuda")
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())

    def step():
        out = spnn.embedding(table, t, 0.5)
        return out, torch.autograd.grad(out, table, dy)[0]
    with torch.cuda.stream(stream):
        step()
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            out, grad = step()
    torch.cuda.synchronize()
    for _ in range(3):
        t.copy_(torch.randint(0, 500, (700,), device="cuda"))
        dy.copy_(torch.randn_like(dy))
        graph.replay()
        torch.cuda.synchronize()
        want = step()
        assert torch.equal(out, want[0]) and torch.equal(grad, want[1])


def test_refusals(gpu_handle):
    import torch
    import mluop_hip
    table, t = torch.zeros(4, 8, device="cuda"), torch.zeros(3, dtype=torch.int32, device="cuda")
    for args in ((table.double(), t), (table[0], t), (table, t.short()), (table, t.cpu()), (table.cpu(), t)):
        with pytest.raises(ValueError):
            mluop_hip.embedding_forward(gpu_handle, *args)
    grad = torch.zeros(3, 8, device="cuda")
    for args in ((grad[:2], t, 4), (grad.double(), t, 4), (grad, t.cpu(), 4)):
        with pytest.raises(ValueError):
            mluop_hip.embedding_backward(gpu_handle, *args)
    with pytest.raises(mluop_hip.MluOpError):
        mluop_hip.embedding_backward(gpu_handle, grad, t, 0)
