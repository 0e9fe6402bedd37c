"""AdamW over many tensors: against the formula in float64 at sizes around a thread, a state block, a workgroup and a launch,
at every pair of types, with views that are not aligned; 8-bit states as codes and scales; the optimizer against
torch.optim.AdamW, with steps that miss gradients, saved states and strided parameters."""
import math

import pytest

pytestmark = pytest.mark.gpu

HYPER = dict(lr=2e-3, betas=(0.9, 0.95), eps=1e-8, weight_decay=0.03)
U = 2.0 ** -24  # half a unit in the last place of fp32, relative


def reference(p, g, m, v, step, lr, betas, eps, weight_decay, grad_scale=1.0):
    """(p, m, v) after a step, and what fp32 roundings may add to p, in float64"""
    import torch
    p, g, m, v = (t.double() for t in (p, g, m, v))
    g = g * grad_scale
    m1 = betas[0] * m + (1 - betas[0]) * g
    v1 = betas[1] * v + (1 - betas[1]) * g * g
    move = lr / (1 - betas[0] ** step) * m1 / (torch.sqrt(v1 / (1 - betas[1] ** step)) + eps)
    p1 = p * (1 - lr * weight_decay) - move
    # p: two roundings of the product and one of the difference.  The step: its two factors as floats, those of m (which may
    # cancel), root, reciprocal (one unit each) and the products around them: twenty halves of a unit cover them
    m_terms = betas[0] * m.abs() + (1 - betas[0]) * g.abs()
    room = 3 * U * (p.abs() + move.abs()) + 20 * U * move.abs() * torch.where(m1 != 0, m_terms / m1.abs(), 1.0)
    return p1, m1, v1, room, 5 * U * m_terms


def tensors(sizes, dtype, grad_dtype, master, skew, seed):
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)

    def flat(n, scale, as_type, offset=0):
        t = (torch.randn(n + offset, device="cuda", generator=g) * scale).to(as_type)
        return t[offset:]
    params = [flat(n, 0.1, dtype, skew) for n in sizes]
    grads = [flat(n, 1e-2, grad_dtype, skew) for n in sizes]
    for t in grads:   # sizes that a block's largest value dwarfs
        t.mul_(torch.exp(2 * torch.randn(t.shape, device="cuda", generator=g)).to(t.dtype))
    m = [flat(n, 1e-2, torch.float32, skew) for n in sizes]
    v = [flat(n, 1e-2, torch.float32, skew).square_() for n in sizes]
    masters = [p.float() + 1e-4 * flat(p.numel(), 1.0, torch.float32) for p in params] if master else None
    return params, grads, m, v, masters


@pytest.mark.parametrize("dtype,grad,master", [("float32", "float32", False), ("float16", "float16", False),
                                               ("bfloat16", "bfloat16", True), ("bfloat16", "float32", False),
                                               ("float16", "float32", True)])
@pytest.mark.parametrize("skew", [0, 1, 8])
def test_states_in_32_bits(gpu_handle, dtype, grad, master, skew):
    import torch
    import mluop_hip
    print("adamw", dtype, grad, master, skew, flush=True)
    dtype, grad = getattr(torch, dtype), getattr(torch, grad)
    sizes = [1, 7, 8, 9, 63, 255, 256, 257, 2047, 2048, 2049, 5003, 0, 70000] + [33 + i for i in range(50)]
    params, grads, m, v, masters = tensors(sizes, dtype, grad, master, skew, 11 + skew)
    want = [reference(*a, 3, **HYPER, grad_scale=0.5) for a in zip(masters or params, grads, m, v)]
    mluop_hip.AdamWTensors(params, m, v, masters).step(gpu_handle, grads, 3, grad_scale=0.5, **HYPER)
    # one rounding of the parameters themselves
    last = {torch.float32: 0.0, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}[dtype]
    for i, (p1, m1, v1, room, m_room) in enumerate(want):
        assert bool(((m[i].double() - m1).abs() <= m_room + 1e-38).all())
        assert bool(((v[i].double() - v1).abs() <= 6 * U * v1 + 1e-38).all())
        if masters:
            assert bool(((masters[i].double() - p1).abs() <= room).all())
            assert torch.equal(params[i], masters[i].to(dtype))
        else:
            assert bool(((params[i].double() - p1).abs() <= room + last * (p1.abs() + room) + 2.0 ** -25).all())


def quantized(m, r):
    """m and r (padded to whole blocks) -> codes and scales by the definition, in float32 where the library's are"""
    import torch
    out = []
    for x, root in ((m, False), (r, True)):
        n = x.numel()
        x = torch.nn.functional.pad(x, (0, -n % 256)).view(-1, 256)
        most = x.abs().amax(dim=1, keepdim=True)
        q = (x * torch.where(most > 1e-30, 448.0 / most, torch.zeros_like(most))).to(torch.float8_e4m3fn).float()
        if root:
            q = torch.where((q == 0) & (x > 0), torch.full_like(q, 2.0 ** -9), q)
        out += [q.view(-1)[:n].to(torch.float8_e4m3fn), (most * (1.0 / 448.0)).view(-1)]
    return out


@pytest.mark.parametrize("dtype,master", [("float32", False), ("bfloat16", False), ("float16", True)])
@pytest.mark.parametrize("skew", [0, 1])
def test_states_in_8_bits(gpu_handle, dtype, master, skew):
    import torch
    import mluop_hip
    print("adamw 8", dtype, master, skew, flush=True)
    dtype = getattr(torch, dtype)
    sizes = [1, 7, 255, 256, 257, 511, 2048, 2049, 70001] + [600 + 7 * i for i in range(60)]
    params, grads, m, v, masters = tensors(sizes, dtype, dtype, master, skew, 5)
    if sizes[-1] > 0:   # a block of zeros, one without gradients, a tiny value beside a large one
        grads[4].zero_()
        m[4].zero_()
        v[4].zero_()
        v[6][3], v[6][4] = 1e4, 1e-12
    states = [quantized(a, b.sqrt()) for a, b in zip(m, v)]
    mq, ms, rq, rs = ([s[k].clone() for s in states] for k in range(4))

    def held(q, s):
        return q.float() * s.repeat_interleave(256)[:q.numel()]
    want = [reference(p, g, held(s[0], s[1]), held(s[2], s[3]) ** 2, 5, **HYPER)
            for p, g, s in zip(masters or params, grads, states)]
    if skew:
        mq = [torch.cat([q.view(torch.uint8)[:1], q.view(torch.uint8)])[1:].view(torch.float8_e4m3fn) for q in mq]
    mluop_hip.AdamWTensors(params, mq, rq, masters, ms, rs).step(gpu_handle, grads, 5, **HYPER)
    last = {torch.float32: 0.0, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}[dtype]
    for i, (p1, m1, v1, room, m_room) in enumerate(want):
        got = masters[i] if masters else params[i]
        slack = 0.0 if masters else last * (p1.abs() + room) + 2.0 ** -25
        # (the root of a v that was squared: two more roundings of the denominator, inside the twenty)
        assert bool(((got.double() - p1).abs() <= room + slack).all()), sizes[i]
        for q, s, x, x_room in ((mq[i], ms[i], m1, m_room), (rq[i], rs[i], v1.sqrt(), 5 * U * v1.sqrt())):
            blocks = torch.nn.functional.pad(x.abs(), (0, -x.numel() % 256)).view(-1, 256)
            most = blocks.amax(dim=1)
            assert bool(((s.double() * 448 - most).abs() <= 8 * U * most + 5 * U * blocks.amax(dim=1)
                         + x_room.max() * (most > 0)).all())
            unit = s.double().repeat_interleave(256)[:x.numel()]
            # half of a code's own step (three bits of mantissa, least step 2^-9), and up to one for the least code of a root
            off = (q.double() * unit - x).abs()
            step = torch.maximum(x.abs() * 2.0 ** -4, unit * 2.0 ** -10) * (1 + 1e-5) + x_room
            if q is rq[i]:
                tiny = (x > 0) & (x <= unit * 2.0 ** -9)
                step = torch.where(tiny, unit * 2.0 ** -9, step)
                assert bool((q.float()[(x > 0) & (unit > 0)] > 0).all())
            assert bool((off <= step).all()), sizes[i]


def test_blocks_of_nothing(gpu_handle):
    """zero gradients on zero states: only the decay is left, and no NaN comes from a scale of zero"""
    import torch
    import mluop_hip
    p = torch.randn(1000, device="cuda")
    was = p.clone()
    q = [torch.zeros(1000, dtype=torch.uint8, device="cuda") for _ in range(2)]
    s = [torch.zeros(4, device="cuda") for _ in range(2)]
    plan = mluop_hip.AdamWTensors([p], [q[0]], [q[1]], None, [s[0]], [s[1]])
    plan.step(gpu_handle, [torch.zeros_like(p)], 1, **HYPER)
    assert torch.allclose(p, was * (1 - HYPER["lr"] * HYPER["weight_decay"]), rtol=1e-6, atol=0)
    assert not bool(q[0].any() | q[1].any()) and not bool((s[0] != 0).any() | (s[1] != 0).any())
    plan.step(gpu_handle, [None], 2, **HYPER)   # (nothing to do)


def test_a_large_tensor(gpu_handle):
    """offsets of more than 31 bits in bytes and elements of the parameters"""
    import torch
    import mluop_hip
    n = (1 << 31) + 1000
    p = torch.zeros(n, dtype=torch.bfloat16, device="cuda")
    g = torch.zeros(n, dtype=torch.bfloat16, device="cuda")
    g[-1000:] = torch.linspace(-1, 1, 1000, device="cuda").to(torch.bfloat16)
    q = [torch.zeros(n, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn) for _ in range(2)]
    s = [torch.zeros(-(-n // 256), device="cuda") for _ in range(2)]
    mluop_hip.AdamWTensors([p], [q[0]], [q[1]], None, [s[0]], [s[1]]).step(gpu_handle, [g], 1, **HYPER)
    tail = g[-1000:].float()
    want = -HYPER["lr"] * tail / (tail.abs() + HYPER["eps"])
    assert torch.allclose(p[-1000:].float(), torch.where(tail == 0, 0.0, want), rtol=2.0 ** -7, atol=1e-12)
    assert not bool(p[:1000].any()) and not bool(p[(1 << 31) - 100000:1 << 31].any())


def test_repeats_bit_by_bit(gpu_handle):
    import torch
    import mluop_hip
    sizes = [100, 5000, 33]
    got = []
    for _ in range(2):
        params, grads, m, v, _ = tensors(sizes, torch.float32, torch.float32, False, 0, 2)
        plan = mluop_hip.AdamWTensors(params, m, v)
        for step in (1, 2, 3):
            plan.step(gpu_handle, grads, step, **HYPER)
        got.append(torch.cat(params + m + v))
    assert torch.equal(got[0], got[1])


@pytest.mark.parametrize("bits", [32, 8])
def test_optimizer_learns_as_torch_does(bits):
    import torch
    from mluop_hip.optim import AdamW

    def train(make):
        torch.manual_seed(3)
        net = torch.nn.Sequential(torch.nn.Linear(33, 130), torch.nn.SiLU(), torch.nn.Linear(130, 5)).cuda()
        x, y = torch.randn(200, 33, device="cuda"), torch.randn(200, 5, device="cuda")
        opt, losses = make(net.parameters()), []
        for _ in range(30):
            opt.zero_grad()
            loss = (net(x) - y).square().mean()
            loss.backward()
            opt.step()
            losses.append(float(loss))
        return torch.cat([p.detach().flatten() for p in net.parameters()]), losses, opt
    hyper = dict(lr=3e-3, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.01)
    want, ref_losses, _ = train(lambda ps: torch.optim.AdamW(ps, **hyper))
    got, losses, opt = train(lambda ps: AdamW(ps, state_bits=bits, **hyper))
    if bits == 32:
        assert float((got - want).abs().max()) < 1e-4
    else:   # (only the first layer's weight is large enough for 8 bits)
        kinds = [("exp_avg_scale" in s) for s in opt.state.values()]
        assert kinds == [True, False, False, False]
        assert losses[-1] < 1.05 * ref_losses[-1] + 1e-3 and losses[-1] < 0.9 * losses[0]


def test_optimizer_state_is_saved_and_goes_on():
    import torch
    from mluop_hip.optim import AdamW

    def make():
        torch.manual_seed(0)
        ps = [torch.nn.Parameter(torch.randn(n, device="cuda").to(torch.bfloat16)) for n in (10, 9000)]
        ps.append(torch.nn.Parameter(torch.randn(64, 100, device="cuda").to(torch.bfloat16).t()))   # columns first
        return ps, AdamW(ps, state_bits=8, master_weights=True, lr=1e-2)

    def grads(ps, k):
        g = torch.Generator(device="cuda").manual_seed(k)
        for i, p in enumerate(ps):
            p.grad = torch.randn(p.shape, device="cuda", generator=g).to(p.dtype)
            if k == 1 and i == 0:
                p.grad = None   # (its step count falls behind)
    a, opt_a = make()
    for k in range(4):
        grads(a, k)
        opt_a.step(grad_scale=0.5)
    assert opt_a.state[a[0]]["step"] == 3 and opt_a.state[a[1]]["step"] == 4
    b, opt_b = make()
    for k in range(2):
        grads(b, k)
        opt_b.step(grad_scale=0.5)
    c, opt_c = make()
    for p, q in zip(c, b):
        p.data.copy_(q.data)
    opt_c.load_state_dict(opt_b.state_dict())
    assert opt_c.state[c[1]]["exp_avg"].dtype == torch.float8_e4m3fn
    assert opt_c.state[c[1]]["master"].dtype == torch.float32
    for k in (2, 3):
        grads(c, k)
        opt_c.step(grad_scale=0.5)
    for p, q in zip(a, c):
        assert torch.equal(p, q)


def test_refusals(gpu_handle):
    import torch
    import mluop_hip

    def t(n, dtype=torch.float32):
        return torch.zeros(n, dtype=dtype, device="cuda")
    make = mluop_hip.AdamWTensors
    for args in (([t(4)], [t(4)], []), ([t(4)], [t(5)], [t(4)]), ([t(4, torch.int32)], [t(4)], [t(4)]),
                 ([t(4)], [t(4, torch.float16)], [t(4)]), ([t(4)], [t(4)], [t(4)], [t(4)]),
                 ([t(4), t(4, torch.float16)], [t(4)] * 2, [t(4)] * 2), ([t(8)[::2]], [t(4)], [t(4)]),
                 ([torch.zeros(4)], [t(4)], [t(4)]),
                 ([t(257)], [t(257, torch.uint8)], [t(257, torch.uint8)], None, [t(1)], [t(2)])):
        with pytest.raises(ValueError):
            make(*args)
    plan = make([t(4)], [t(4)], [t(4)])
    for grads in ([], [t(5)], [t(4, torch.float16)]):
        with pytest.raises(ValueError):
            plan.step(gpu_handle, grads, 1, **HYPER)
    for more in (dict(step=0), dict(step=1, betas=(1.0, 0.9)), dict(step=1, eps=-1.0), dict(step=1, lr=math.nan)):
        with pytest.raises(mluop_hip.MluOpError):
            plan.step(gpu_handle, [t(4)], **{**HYPER, **more})


def test_codes_are_those_of_plain_operations(gpu_handle):
    """half a code on, one unit in the last place decides between two of them: codes and scales of two steps are the same as
    of torch's operations, one after the other, in fp32"""
    import torch
    import mluop_hip
    n, beta1, beta2, lr, eps = 8_000_000, 0.9, 0.95, 1e-3, 1e-8
    g = torch.Generator(device="cuda").manual_seed(77)
    master = torch.randn(n, device="cuda", generator=g) * 0.05
    param, want = master.bfloat16(), master.clone()
    m, v = (torch.zeros(n, dtype=torch.uint8, device="cuda") for _ in range(2))
    ms, vs = (torch.zeros(n // 256, device="cuda") for _ in range(2))
    plan = mluop_hip.AdamWTensors([param], [m], [v], [master], [ms], [vs])

    def codes(x, root):
        x = x.view(-1, 256)
        most = x.abs().amax(dim=1, keepdim=True)
        q = (x * (most.reciprocal() * 448.0)).to(torch.float8_e4m3fn)
        if root:
            f = q.float()
            q = torch.where((f == 0) & (x > 0), torch.full_like(f, 2.0 ** -9), f).to(torch.float8_e4m3fn)
        return q.view(-1), most.view(-1) * (1.0 / 448.0)

    def values(q, scale):
        return (q.float().view(-1, 256) * scale.unsqueeze(1)).view(-1)

    mine = [torch.zeros(n, device="cuda").to(torch.float8_e4m3fn) for _ in range(2)]
    scales = [torch.zeros(n // 256, device="cuda") for _ in range(2)]
    for step in (1, 2):
        grad = (torch.randn(n, device="cuda", generator=g) * 1e-2).bfloat16()
        plan.step(gpu_handle, [grad], step, lr, (beta1, beta2), eps, 0.0)
        d = grad.float()
        a = values(mine[0], scales[0]) * beta1 + d * (1.0 - beta1)
        r = torch.sqrt(values(mine[1], scales[1]).square() * beta2 + d * d * (1.0 - beta2))
        want = want - lr / (1.0 - beta1 ** step) * (a / (r * (1.0 / (1.0 - beta2 ** step) ** 0.5) + eps))
        (mine[0], scales[0]), (mine[1], scales[1]) = codes(a, False), codes(r, True)
        for got, scale, q, s in ((m, ms, mine[0], scales[0]), (v, vs, mine[1], scales[1])):
            assert torch.equal(got.view(torch.float8_e4m3fn).float(), q.float()) and torch.equal(scale, s)
        assert float((master - want).abs().max()) < 1e-6 * step
