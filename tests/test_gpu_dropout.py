"""Dropout onto a residual: the generator against its published words, masks element by element, gradients, shares of what is kept,
counts of calls across replays of a graph; refusals."""
import pytest

LAST = {"float32": 2.0 ** -24, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}


def test_the_reference_has_the_published_words():
    """the known answers that come with the generator's publication"""
    import numpy as np
    from philox_reference import words
    ones = 0xFFFFFFFF
    for counter, key, want in (
            ([0] * 4, [0] * 2, [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]),
            ([ones] * 4, [ones] * 2, [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]),
            ([0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344], [0xA4093822, 0x299F31D0],
             [0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1])):
        assert words(np.array(counter), key).tolist() == want


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("n", [1, 7, 8, 9, 4095, 4096, 4097, 100_003])
@pytest.mark.parametrize("p", [0.1, 0.5])
@pytest.mark.parametrize("add", [False, True])
def test_against_the_mask(gpu_handle, dtype, n, p, add):
    import torch
    import mluop_hip
    from philox_reference import kept
    kind = getattr(torch, dtype)
    g = torch.Generator(device="cuda").manual_seed(n)
    x = torch.randn(n, device="cuda", generator=g).to(kind)
    r = torch.randn(n, device="cuda", generator=g).to(kind) if add else None
    for seed, call in ((0, 0), (-3, 5), (1 << 62, (1 << 40) + 7), (12345, -1)):
        state = torch.tensor([seed, call], device="cuda")
        mask, scale = kept(n, p, seed, call)
        mask = torch.from_numpy(mask).cuda()
        got = mluop_hip.dropout_add_forward(gpu_handle, x, r, p, state)
        want = torch.where(mask, x.double() * scale, 0.0) + (r.double() if add else 0.0)
        # (the factor and the sum have a rounding each in fp32, and the result one)
        room = LAST[dtype] * want.abs() + 2.0 ** -23 * (x.double().abs() * scale + want.abs()) + 2.0 ** -25
        assert bool(((got.double() - want).abs() <= room).all())
        if not add:
            assert torch.equal(got != 0, mask & (x != 0))
        assert torch.equal(mluop_hip.dropout_add_backward(gpu_handle, x, p, state),
                           mluop_hip.dropout_add_forward(gpu_handle, x, None, p, state))


@pytest.mark.gpu
@pytest.mark.parametrize("n", [17, 50_000])
def test_ends_of_the_range(gpu_handle, n):
    """nothing dropped, everything dropped, and what is dropped does not count"""
    import torch
    import mluop_hip
    x, r = torch.randn(n, device="cuda"), torch.randn(n, device="cuda")
    x[3], x[9] = float("nan"), float("inf")
    state = torch.tensor([7, 8], device="cuda")
    assert torch.equal(mluop_hip.dropout_add_forward(gpu_handle, x, None, 0.0, state).nan_to_num(5.0), x.nan_to_num(5.0))
    assert torch.equal(mluop_hip.dropout_add_forward(gpu_handle, x, None, 2.0 ** -18, state).nan_to_num(5.0), x.nan_to_num(5.0))
    assert torch.equal(mluop_hip.dropout_add_forward(gpu_handle, x, r, 1.0, state), r)
    assert not bool(mluop_hip.dropout_add_forward(gpu_handle, x, None, 1.0, state).any())


@pytest.mark.gpu
def test_shares(gpu_handle):
    """of four million elements a share of p is dropped, to five standard deviations; calls and seeds differ"""
    import torch
    import mluop_hip
    n = 1 << 22
    x = torch.ones(n, device="cuda")
    masks = []
    for seed, call in ((1, 0), (1, 1), (2, 0)):
        for p in (0.02, 0.3):
            out = mluop_hip.dropout_add_forward(gpu_handle, x, None, p, torch.tensor([seed, call], device="cuda"))
            share = float((out == 0).double().mean())
            assert abs(share - p) <= 5 * (p * (1 - p) / n) ** 0.5 + 2.0 ** -17
        masks.append(out == 0)
    for a, b in ((0, 1), (0, 2), (1, 2)):
        both = float((masks[a] & masks[b]).double().mean())
        assert abs(both - 0.09) <= 5 * (0.09 * 0.91 / n) ** 0.5 + 2.0 ** -16


@pytest.mark.gpu
def test_shapes_views_and_addresses(gpu_handle):
    import torch
    import mluop_hip
    state = torch.tensor([3, 4], device="cuda")
    x, r = torch.randn(60, 24, device="cuda").half(), torch.randn(60, 24, device="cuda").half()
    want = mluop_hip.dropout_add_forward(gpu_handle, x, r, 0.3, state)
    flat = torch.zeros(60 * 24 + 1, dtype=torch.float16, device="cuda")
    wide = torch.zeros(60, 50, dtype=torch.float16, device="cuda")
    for view in (flat[1:].view(60, 24), wide[:, 5:29], torch.empty(24, 60, dtype=torch.float16, device="cuda").t()):
        view.copy_(x)
        assert torch.equal(mluop_hip.dropout_add_forward(gpu_handle, view, r, 0.3, state), want)
        view.copy_(r)
        assert torch.equal(mluop_hip.dropout_add_forward(gpu_handle, x, view, 0.3, state), want)
    assert torch.equal(mluop_hip.dropout_add_forward(gpu_handle, x.view(5, 12, 24), r.view(5, 12, 24), 0.3, state), want.view(5, 12, 24))
    assert mluop_hip.dropout_add_forward(gpu_handle, x[:0], r[:0], 0.3, state).shape == (0, 24)


@pytest.mark.gpu
def test_autograd_and_module():
    import torch
    from mluop_hip import nn as spnn
    torch.manual_seed(4)
    layer = spnn.DropoutAdd(0.25).cuda()
    seed = int(layer.state[0])
    x, r = (torch.randn(300, 40, device="cuda", requires_grad=True) for _ in range(2))
    out, again = layer(x, r), layer(x, r)
    assert layer.state.tolist() == [seed, 2] and not torch.equal(out, again)
    dy = torch.randn_like(x)
    dx, dr = torch.autograd.grad(out, [x, r], dy)
    mask = (out - r).detach().abs() > 1e-4 * (1 + r.detach().abs())
    scale = 65536 / (65536 - 16384)
    clear = x.detach().abs() > 1e-2
    assert torch.equal(dr, dy)
    assert torch.allclose(dx[clear], torch.where(mask, dy * scale, torch.zeros_like(dy))[clear], rtol=2.0 ** -22)
    state = torch.tensor([seed, 0], device="cuda")   # (the call's number is that from before the call)
    assert torch.equal(spnn.dropout_add(x, r, 0.25, state), out)
    out = spnn.dropout_add(x, r, 0.25, state)
    state.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.sum().backward()
    saved = spnn.DropoutAdd(0.25, seed=1).cuda()
    saved.load_state_dict(layer.state_dict())
    assert torch.equal(saved(x, r), layer(x, r))
    layer.eval()
    count = layer.state.tolist()
    assert torch.equal(layer(x, r), x + r) and layer(x) is x and layer.state.tolist() == count
    with pytest.raises(ValueError):
        spnn.DropoutAdd(1.5)


@pytest.mark.gpu
def test_every_replay_drops_other_elements():
    import torch
    from mluop_hip import nn as spnn
    layer, twin = spnn.DropoutAdd(0.4, seed=9).cuda(), spnn.DropoutAdd(0.4, seed=9).cuda()
    x, r = torch.randn(5000, 16, device="cuda").bfloat16(), torch.randn(5000, 16, device="cuda").bfloat16()
    dy = torch.randn_like(x)

    def step(layer):
        leaves = [t.detach().requires_grad_() for t in (x, r)]
        out = layer(*leaves)
        return [out] + list(torch.autograd.grad(out, leaves, dy))
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step(layer)
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            out = step(layer)
    torch.cuda.synchronize()
    step(twin)
    for _ in range(4):
        x.copy_(torch.randn_like(x))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, step(twin)))
        assert layer.state.tolist() == twin.state.tolist()


@pytest.mark.gpu
def test_refusals(gpu_handle):
    import torch
    import mluop_hip
    x, state = torch.randn(10, 8, device="cuda"), torch.tensor([1, 2], device="cuda")
    for bad in (dict(features=x.double()), dict(features=x.cpu()), dict(residual=x[:5]), dict(residual=x.half()),
                dict(p=-0.1), dict(p=1.1), dict(p=float("nan")), dict(state=state.int()), dict(state=state.cpu()),
                dict(state=state[:1]), dict(residual=x.cpu())):
        with pytest.raises(ValueError):
            mluop_hip.dropout_add_forward(gpu_handle, **{**dict(features=x, residual=x, p=0.5, state=state), **bad})
