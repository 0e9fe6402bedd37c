"""GroupNormAct on sparse tensors whose rows lie in any order: the statistics are those of each sample's rows, wherever they
are; what is known about the order, and indice_keys that read like the norm's own."""
import pytest

pytestmark = pytest.mark.gpu


def tensor(shuffle, seed=0, channels=16, samples=3, **kw):
    import torch
    from mluop_hip import nn as spnn
    idx = torch.tensor([[n, 0, i // 20, i % 20] for n in range(samples) for i in range(60 + 50 * n)], dtype=torch.int32,
                       device="cuda")
    g = torch.Generator(device="cuda").manual_seed(seed)
    feats = torch.randn(idx.shape[0], channels, device="cuda", generator=g)
    perm = torch.randperm(idx.shape[0], generator=g, device="cuda") if shuffle else torch.arange(idx.shape[0], device="cuda")
    return spnn.SparseTensor(feats[perm].requires_grad_(), idx[perm], (1, 20, 20), samples, distinct=True, **kw), perm


def expected(feats, samples, norm):
    """every sample's rows by torch's group norm"""
    import torch
    out = torch.empty_like(feats)
    for n in samples.unique():
        rows = (samples == n).nonzero()[:, 0]
        z = torch.nn.functional.group_norm(feats[rows].t()[None], norm.groups, norm.weight, norm.bias, norm.eps)[0].t()
        out[rows] = torch.nn.functional.silu(z)
    return out


@pytest.mark.parametrize("shuffle", [False, True])
def test_rows_in_any_order(shuffle):
    import torch
    from mluop_hip import nn as spnn
    torch.manual_seed(1)
    x, _ = tensor(shuffle)
    norm = spnn.GroupNormAct(4, 16, activation="silu").cuda()
    with torch.no_grad():
        norm.weight.normal_(1, 0.3)
        norm.bias.normal_(0, 0.3)
    got = norm(x).features
    want = expected(x.features, x.indices[:, 0], norm)
    assert torch.allclose(got, want, atol=1e-5)
    dy = torch.randn_like(got)
    inputs = [x.features, norm.weight, norm.bias]
    for a, b in zip(torch.autograd.grad(got, inputs, dy), torch.autograd.grad(want, inputs, dy)):
        assert torch.allclose(a, b, rtol=1e-3, atol=1e-3 * float(b.abs().max()))


@pytest.mark.parametrize("shuffle", [False, True])
def test_in_a_network(shuffle):
    """behind submanifold layers rows keep their order, behind a strided one they come in order, behind its inverse as before"""
    import torch
    from mluop_hip import nn as spnn
    torch.manual_seed(2)
    net = spnn.SparseSequential(
        spnn.SubMConv3d(16, 32, 3), spnn.GroupNormAct(8, 32, activation="silu"),
        spnn.SparseConv3d(32, 32, 3, stride=2, padding=1, indice_key="down"), spnn.GroupNormAct(8, 32, activation="silu"),
        spnn.SparseInverseConv3d(32, 16, 3, indice_key="down"), spnn.GroupNormAct(4, 16, activation="silu")).cuda()
    x, _ = tensor(shuffle)
    y = x
    for conv, norm in zip(list(net)[::2], list(net)[1::2]):
        y = conv(y)
        y = y.replace_features(expected(y.features, y.indices[:, 0], norm))
    fresh, _ = tensor(shuffle)
    got = net(fresh)
    assert torch.equal(got.indices, y.indices) and torch.allclose(got.features, y.features, atol=1e-4)


def test_row_starts_of_rows_in_no_order_are_refused():
    x, _ = tensor(True)
    with pytest.raises(ValueError):
        x.row_starts()
    assert tensor(False)[0].row_starts().tolist() == [0, 60, 170, 330]


def test_samples_without_rows_and_rows_of_no_sample():
    import torch
    from mluop_hip import nn as spnn
    x, _ = tensor(True)
    wide = spnn.SparseTensor(x.features, x.indices, x.spatial_shape, 5, distinct=True)
    few = spnn.SparseTensor(x.features, x.indices, x.spatial_shape, 2, distinct=True)
    norm = spnn.GroupNormAct(4, 16, activation="silu").cuda()
    want = expected(x.features, x.indices[:, 0], norm)
    assert torch.allclose(norm(wide).features, want, atol=1e-5)
    outside = x.indices[:, 0] >= 2
    got = norm(few).features
    assert torch.allclose(got[~outside], want[~outside], atol=1e-5) and not bool(got[outside].any())


@pytest.mark.parametrize("key", ["row_starts", "samples"])
def test_indice_keys_of_any_name(key):
    import torch
    from mluop_hip import nn as spnn
    torch.manual_seed(3)
    net = spnn.SparseSequential(spnn.GroupNormAct(4, 16), spnn.SubMConv3d(16, 16, 3, indice_key=key),
                                spnn.GroupNormAct(4, 16), spnn.SubMConv3d(16, 16, 3, indice_key=key)).cuda()
    x, _ = tensor(False)
    got = net(x).features
    for m in net:
        if isinstance(m, spnn.SubMConv3d):
            m.indice_key = "another"
    assert torch.equal(got, net(tensor(False)[0]).features)
    y = tensor(False)[0]
    net[0](y)
    assert key not in y.rulebooks


def test_the_order_is_looked_at_once_and_not_where_it_is_given(monkeypatch):
    import torch
    from mluop_hip import nn as spnn
    import mluop_hip
    monkeypatch.setattr(mluop_hip, "GUARD_BYTES", 0)
    looked = []
    real = spnn._in_sample_order
    monkeypatch.setattr(spnn, "_in_sample_order", lambda samples: looked.append(1) or real(samples))
    norm = spnn.GroupNormAct(4, 16).cuda()
    for shuffle in (False, True):
        x, _ = tensor(shuffle)
        norm(norm(norm(x)))
        norm(x.replace_features(x.features * 2))
        assert len(looked) == 1
        looked.clear()
    x, _ = tensor(False, ordered=True)
    down = spnn.SparseConv3d(16, 16, 3, stride=2, padding=1).cuda()
    norm(down(norm(x)))
    norm(down(tensor(True)[0]))   # (a strided layer's rows are in order)
    one, _ = tensor(True, samples=1)
    norm(one)
    assert not looked


def test_a_word_that_is_not_true_is_refused_behind_guard_bands(gpu_handle):
    from mluop_hip import nn as spnn
    norm = spnn.GroupNormAct(4, 16).cuda()
    norm(tensor(False, ordered=True)[0])
    with pytest.raises(ValueError, match="ordered"):
        norm(tensor(True, ordered=True)[0])


def test_captured():
    """nothing is waited for while a graph is captured: the order is given, or has been looked at"""
    import torch
    from mluop_hip import nn as spnn
    norm = spnn.GroupNormAct(4, 16, activation="silu").cuda()
    stream = torch.cuda.Stream()
    for kind in ("looked", "given"):
        x, _ = tensor(kind == "looked", ordered=None if kind == "looked" else True)
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream), torch.no_grad():
            if kind == "looked":
                norm(x)
            norm(tensor(False)[0])
            stream.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                out = norm(x).features
        torch.cuda.synchronize()
        for k in range(3):
            with torch.no_grad():
                x.features.copy_(torch.randn_like(x.features))
            graph.replay()
            torch.cuda.synchronize()
            with torch.no_grad():
                assert torch.equal(out, norm(x).features)


def test_refused_while_capturing(monkeypatch):
    """(no capture is begun: what asks whether one is answers that it is)"""
    from mluop_hip import nn as spnn
    monkeypatch.setattr(spnn, "_capturing", lambda: True)
    x, _ = tensor(False)
    with pytest.raises(RuntimeError, match="ordered"):
        spnn.GroupNormAct(4, 16).cuda()(x)
