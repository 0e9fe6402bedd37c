"""The operators of a residual block as they are used together: norm, recurrence both ways, dropout onto the residual, norm, experts,
dropout; against the formulas in float64, captured into a graph, and in the example."""
import importlib.util
import os

import pytest

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def example():
    spec = importlib.util.spec_from_file_location("voxel_sequence", os.path.join(ROOT, "examples", "voxel_sequence.py"))
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def cells(sizes):
    import torch
    return torch.tensor([[n, 0, i // 20, i % 20] for n, size in enumerate(sizes) for i in range(size)], dtype=torch.int32, device="cuda")


def scan(layer, x, starts):
    """the recurrence layer row by row"""
    import torch
    features, gates = (x @ layer.into.weight.t() + layer.into.bias).chunk(2, dim=1)
    rows = [None] * x.shape[0]
    for lo, hi in zip(starts, starts[1:]):
        h = torch.zeros_like(features[0])
        for t in (range(hi - 1, lo - 1, -1) if layer.reverse else range(lo, hi)):
            a = torch.sigmoid(gates[t])
            h = rows[t] = (a * h + (1 - a) * features[t]) if layer.kind == "sigmoid" else a * h + features[t]
    return torch.stack(rows) @ layer.back.weight.t() + layer.back.bias


def experts(layer, x):
    import torch
    scores = x @ layer.gate.weight.t()
    top, chosen = torch.topk(scores, layer.choices, dim=1)
    weight = torch.zeros_like(scores).scatter(1, chosen, torch.softmax(top, dim=1))
    return sum(weight[:, e:e + 1] * (torch.nn.functional.silu(x @ layer.up.weight[e]) @ layer.down.weight[e])
               for e in range(layer.experts))


def dropped(x, p, state):
    import torch
    from philox_reference import kept
    mask, scale = kept(x.numel(), p, *state)
    return x * (torch.from_numpy(mask).view(x.shape).to(x) * scale)


@pytest.mark.parametrize("kind", ["sigmoid", "exp"])
def test_block_against_the_formulas(kind):
    """(exp: the layer's decay is exp(-softplus(-gate)), which is a sigmoid)"""
    import copy
    import torch
    from mluop_hip import nn as spnn
    torch.manual_seed(1)
    block = example().Block(32, kind, experts=5, dropout=0.25).cuda()
    sizes, starts = (30, 25, 41), [0, 30, 55, 96]
    x = torch.randn(96, 32, device="cuda", requires_grad=True)
    states = [layer.state.tolist() for layer in block.residuals]
    got = block(spnn.SparseTensor(x, cells(sizes), (1, 20, 20), 3, distinct=True)).features
    twin = copy.deepcopy(block).double().cpu()
    y = x.detach().double().cpu().requires_grad_()

    def norm(layer, v):
        return torch.nn.functional.layer_norm(v, (32,), layer.weight, layer.bias, layer.eps)
    first = norm(twin.norms[0], y)
    mixed = scan(twin.mix.forwards, first, starts) + scan(twin.mix.backwards, first, starts)
    middle = y + dropped(mixed, 0.25, states[0])
    want = middle + dropped(experts(twin.experts, norm(twin.norms[1], middle)), 0.25, states[1])
    # (a dozen products of 32 to 64 terms in fp32 behind one another, of values of a few units)
    assert float((got.double().cpu() - want).abs().max()) <= 1e-4
    dy = torch.randn_like(got)
    names = ["x"] + [n for n, _ in block.named_parameters()]
    have = torch.autograd.grad(got, [x] + list(block.parameters()), dy)
    ref = torch.autograd.grad(want, [y] + list(twin.parameters()), dy.double().cpu())
    for name, a, b in zip(names, have, ref):
        assert float((a.double().cpu() - b).abs().max()) <= 2e-4 * (1 + float(b.abs().max())), name


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_block_captured(dtype):
    """a forward and a backward pass in a graph, replayed between eager ones of a twin: the same results, new masks every time"""
    import copy
    import torch
    from mluop_hip import nn as spnn
    torch.manual_seed(2)
    block = example().Block(64, "sigmoid", experts=4, dropout=0.2).cuda()
    twin = copy.deepcopy(block)
    rows = 3 * 300
    x, dy = (torch.randn(rows, 64, device="cuda").to(getattr(torch, dtype)) for _ in range(2))
    where = cells((300, 300, 300))

    def step(block):
        leaf = x.detach().requires_grad_()
        out = block(spnn.SparseTensor(leaf, where, (1, 20, 20), 3, distinct=True, ordered=True)).features
        return [out] + list(torch.autograd.grad(out, [leaf] + list(block.parameters()), dy))
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step(block)
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            out = step(block)
    torch.cuda.synchronize()
    step(twin)
    seen = []
    for _ in range(3):
        x.copy_(torch.randn_like(x))
        graph.replay()
        torch.cuda.synchronize()
        want = step(twin)
        for a, b in zip(out, want):
            off, size = (a.float() - b.float()).abs(), float(b.float().abs().max())
            # (a row whose two best experts are within rounding of the third may go elsewhere: few do)
            assert float((off > 2.0 ** -5 * size + 1e-4).float().mean()) <= 0.02
        seen.append(block.residuals[0].state.tolist())
        assert seen[-1] == twin.residuals[0].state.tolist()
    assert len({tuple(s) for s in seen}) == 3


def test_example_runs_and_its_gradients_are_slopes():
    import torch
    module = example()
    net, losses = module.train(3, 1500, torch.bfloat16)
    assert len(losses) == 3 and all(v == v and v < 20 for v in losses)
    # in fp32, without dropout and with all experts chosen (a row that goes to another expert is a step in the loss, and the loss has
    # no slope there): the loss along a direction
    net.eval()
    for block in net.blocks:
        block.experts.choices = block.experts.experts
    categories, indices, labels = module.cloud(600, 5)

    def loss():
        return torch.nn.functional.cross_entropy(net(categories, indices, torch.float32), labels)
    for name in ("embed.weight", "blocks.0.mix.backwards.into.weight", "blocks.1.norms.0.bias", "blocks.1.mix.forwards.back.weight",
                 "blocks.0.experts.down.weight", "norm.weight"):
        p = dict(net.named_parameters())[name]
        (grad,) = torch.autograd.grad(loss(), p)
        # along the gradient, so that the slope is large beside the rounding of the losses
        d = grad / grad.norm()
        with torch.no_grad():
            values = []
            h = 2e-2
            for s in (1, -1):
                p.add_(d, alpha=s * h)
                values.append(float(loss().double()))
                p.add_(d, alpha=-s * h)
        slope, want = (values[0] - values[1]) / (2 * h), float(grad.norm())
        # (third derivatives of the loss times h^2 / 6, and 2^-22 / h of rounding)
        assert abs(slope - want) <= 0.1 * want + 1e-4, name
