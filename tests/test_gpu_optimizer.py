"""The AdamW optimizer over its life: copied and pickled, parameters that miss gradients, calls that are refused, parameters whose
memory is laid out anew, gradients that are not finite, roots below the smallest normal number, and autograd's view of what a
step has changed."""
import copy
import io

import pytest

from launches import launched

pytestmark = pytest.mark.gpu

HYPER = dict(lr=1e-2, betas=(0.9, 0.95), eps=1e-8, weight_decay=0.03)


def parameters(seed=0, dtype=None, sizes=(10, 9000, 300)):
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)
    return [torch.nn.Parameter(torch.randn(n, device="cuda", generator=g).to(dtype or torch.float32)) for n in sizes]


def give_gradients(params, seed, missing=()):
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)
    for i, p in enumerate(params):
        grad = torch.randn(p.shape, device="cuda", generator=g).to(p.dtype)
        p.grad = None if i in missing else grad


@pytest.mark.parametrize("way", ["deepcopy", "pickle"])
@pytest.mark.parametrize("bits", [32, 8])
def test_a_copy_goes_on(way, bits):
    import torch
    from mluop_hip.optim import AdamW
    a = parameters()
    opt = AdamW(a, state_bits=bits, **HYPER)
    give_gradients(a, 1)
    opt.step()
    if way == "deepcopy":
        b, twin = copy.deepcopy((a, opt))
    else:
        buffer = io.BytesIO()
        torch.save((a, opt), buffer)
        buffer.seek(0)
        b, twin = torch.load(buffer, weights_only=False)   # (written above)
    for params, o in ((a, opt), (b, twin)):
        give_gradients(params, 2)
        o.step()
    assert twin.param_groups[0]["params"][0] is b[0]
    for p, q in zip(a, b):
        assert p is not q and torch.equal(p, q)


class Counted:
    """the class of checked tensors, counting how many are made"""

    def __init__(self, real):
        self.real, self.made = real, 0

    def __call__(self, *args):
        self.made += 1
        return self.real(*args)


@pytest.mark.parametrize("bits", [32, 8])
def test_parameters_that_miss_gradients_keep_their_plans(bits, monkeypatch):
    """step counts of one group fall apart, and a step checks no tensor anew for that"""
    import torch
    from mluop_hip import optim
    counted = Counted(optim.AdamWTensors)
    monkeypatch.setattr(optim, "AdamWTensors", counted)
    missing = {2: (0,), 3: (1,), 5: (0, 2), 7: (0, 1, 2)}
    a = parameters()
    opt = optim.AdamW(a, state_bits=bits, **HYPER)
    b = parameters()
    each = [optim.AdamW([p], state_bits=bits, **HYPER) for p in b]
    for k in range(10):
        give_gradients(a, k, missing.get(k, ()))
        give_gradients(b, k, missing.get(k, ()))
        if k == 1:
            counted.made = 0
        opt.step()
        if k >= 1:
            assert counted.made == 0, k
        for o in each:
            o.step()
        counted.made = 0
    assert [opt.state[p]["step"] for p in a] == [7, 8, 8]
    for p, q in zip(a, b):
        assert torch.equal(p, q)


def test_a_refused_step_is_not_counted():
    import torch
    import mluop_hip
    from mluop_hip.optim import AdamW
    a, b = parameters(), parameters()
    opt, ref = AdamW(a, **HYPER), AdamW(b, **HYPER)
    for params, o in ((a, opt), (b, ref)):
        give_gradients(params, 1)
        o.step()
    opt.param_groups[0]["lr"] = float("nan")
    with pytest.raises(mluop_hip.MluOpError):
        opt.step()
    opt.param_groups[0]["lr"] = HYPER["lr"]
    assert [opt.state[p]["step"] for p in a] == [1, 1, 1]
    opt.step()
    ref.step()
    for p, q in zip(a, b):
        assert torch.equal(p, q)


@pytest.mark.parametrize("change", ["transposed", "shorter"])
def test_parameters_laid_out_anew_on_the_same_memory(change):
    """the states lie as the parameter did: a step that would mix them up is refused"""
    import torch
    from mluop_hip.optim import AdamW
    p = torch.nn.Parameter(torch.randn(64, 64, device="cuda"))
    opt = AdamW([p], **HYPER)
    p.grad = torch.randn(64, 64, device="cuda")
    opt.step()
    p.data = p.data.t() if change == "transposed" else p.data[:32]
    p.grad = torch.randn(p.shape, device="cuda")
    was = p.detach().clone()
    with pytest.raises(ValueError):
        opt.step()
    assert torch.equal(p, was)


def test_autograd_notices_a_step():
    """a value that a backward pass needs was changed by a step in between"""
    import torch
    from mluop_hip.optim import AdamW
    a = parameters(sizes=(40, 5000))
    idle = torch.nn.Parameter(torch.ones(3, device="cuda"))
    opt = AdamW(a + [idle], state_bits=8, **HYPER)
    give_gradients(a, 1)
    opt.step()
    x = torch.randn(40, device="cuda", requires_grad=True)
    y = (x * a[0]).sum()
    versions = [p._version for p in a + [idle]]
    opt.step()
    assert all(p._version > v for p, v in zip(a, versions)) and idle._version == versions[-1]
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
    # what is made without a record of versions can be stepped too
    with torch.inference_mode():
        q = torch.nn.Parameter(torch.ones(5, device="cuda"), requires_grad=False)
        q.grad = torch.ones(5, device="cuda")
        AdamW([q], **HYPER).step()
    assert bool((q < 1).all())


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_gradients_that_are_not_finite(gpu_handle, bits, bad):
    """a NaN poisons its own element and no other; an infinite one, with 8-bit states, its block of 256, whose scale it is"""
    import torch
    import mluop_hip
    n, at = 1000, 300
    start = parameters(4, sizes=(n,))[0].detach()
    grad = parameters(5, sizes=(n,))[0].detach()
    grad[at] = 0.0
    spoilt = grad.clone()
    spoilt[at] = bad
    got = []
    for g in (grad, spoilt):
        p = start.clone()
        states = [torch.zeros(n, dtype=torch.float32 if bits == 32 else torch.uint8, device="cuda") for _ in range(2)]
        scales = [[torch.zeros(4, device="cuda")] for _ in range(2)] if bits == 8 else [None, None]
        plan = mluop_hip.AdamWTensors([p], states[:1], states[1:], None, *scales)
        plan.step(gpu_handle, [g], 1, **HYPER)
        one = p.clone()
        held = [s.view(torch.float8_e4m3fn).float() if bits == 8 else s.clone() for s in states]
        plan.step(gpu_handle, [grad], 2, **HYPER)
        got.append((one, p, held))
    clean, dirty = got
    block = torch.zeros(n, dtype=torch.bool, device="cuda")
    block[at] = True
    assert torch.equal(dirty[0][~block], clean[0][~block]) and not bool(torch.isfinite(dirty[0][at]))
    for held in dirty[2]:
        assert not bool(torch.isfinite(held[at]))
        if bad != bad:
            assert bool(torch.isnan(held[at]))
    if bits == 8 and bad == bad:
        block[256:512] = True
    # (and so after a step whose gradients are all finite)
    assert not bool(torch.isfinite(dirty[1][at]))
    assert torch.equal(dirty[1][~block], clean[1][~block])
    for a, b in zip(dirty[2], clean[2]):
        assert torch.equal(a[~block], b[~block])


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("size", [1e-18, 1e-19, 1e-20])
def test_roots_of_numbers_below_the_smallest_normal(gpu_handle, bits, size):
    """eps = 0: the first step is lr whatever the gradients' size, also where their squares have few bits left"""
    import torch
    import mluop_hip
    n = 512
    sign = torch.where(torch.arange(n, device="cuda") % 3 == 0, -1.0, 1.0)
    p = torch.zeros(n, device="cuda")
    states = [torch.zeros(n, dtype=torch.float32 if bits == 32 else torch.uint8, device="cuda") for _ in range(2)]
    scales = [[torch.zeros(2, device="cuda")] for _ in range(2)] if bits == 8 else [None, None]
    mluop_hip.AdamWTensors([p], states[:1], states[1:], None, *scales).step(
        gpu_handle, [sign * size], 1, lr=0.5, betas=(0.9, 0.5), eps=0.0, weight_decay=0.0)
    # v = size^2 / 2, a multiple of 2^-149: off by half of that, and its root by half as much relatively
    room = 2.0 ** -149 / size ** 2 + 2.0 ** -20
    assert float((p / (-0.5 * sign) - 1).abs().max()) <= room


def test_an_eps_below_the_smallest_normal(gpu_handle):
    """parameters without gradients so far do not move"""
    import torch
    import mluop_hip
    p = torch.ones(300, device="cuda")
    m, v = torch.zeros(300, device="cuda"), torch.zeros(300, device="cuda")
    mluop_hip.AdamWTensors([p], [m], [v]).step(gpu_handle, [torch.zeros(300, device="cuda")], 1, lr=0.5, betas=(0.9, 0.5),
                                              eps=1e-40, weight_decay=0.0)
    assert bool((p == 1).all())


# Tensors of a launch: what 4 KB of addresses hold.
@pytest.mark.parametrize("bits,master,most", [(32, False, 106), (32, True, 87), (8, False, 74), (8, True, 65)])
@pytest.mark.parametrize("count", ["below", "full", "above", "twice"])
def test_tensors_around_a_launch(gpu_handle, bits, master, most, count):
    """every tensor gets the step it gets alone, however many launches they fill"""
    import torch
    import mluop_hip
    tensors = {"below": most - 1, "full": most, "above": most + 1, "twice": 2 * most + 3}[count]
    g = torch.Generator(device="cuda").manual_seed(tensors)
    sizes = [(37 * i) % 700 + 1 if i % 9 else 2048 * (i // 9 % 3) + 2047 for i in range(tensors)]
    dtype = torch.bfloat16 if master else torch.float32
    params = [torch.randn(n, device="cuda", generator=g).to(dtype) for n in sizes]
    grads = [torch.randn(n, device="cuda", generator=g).to(dtype) for n in sizes]

    def lists(params):
        states = [[torch.zeros(p.numel(), device="cuda") if bits == 32 else
                   torch.zeros(p.numel(), dtype=torch.uint8, device="cuda") for p in params] for _ in range(2)]
        scales = [[torch.zeros(-(-p.numel() // 256), device="cuda") for p in params] for _ in range(2)]
        return (params, *states, [p.float() for p in params] if master else None, *(scales if bits == 8 else (None, None)))
    together, alone = lists([p.clone() for p in params]), lists([p.clone() for p in params])
    plan = mluop_hip.AdamWTensors(*together)
    _, names = launched(gpu_handle, lambda: plan.step(gpu_handle, grads, 1, **HYPER))
    assert names == ["adamwStep"] * (1 if tensors <= most else 2 if tensors <= 2 * most else 3)
    for i in range(tensors):
        mluop_hip.AdamWTensors(*[None if x is None else x[i:i + 1] for x in alone]).step(gpu_handle, grads[i:i + 1], 1, **HYPER)
    for a, b in zip(together, alone):
        if a is not None:
            assert all(torch.equal(x, y) for x, y in zip(a, b))
