"""The operators of a residual block at sizes whose elements, bytes or workgroups pass 32 bits or a launch, and from several
threads and streams at once."""
import threading

import pytest

from test_gpu_launch_limits import handle, room_for  # noqa: F401 (a fixture)

pytestmark = pytest.mark.gpu

EPS = 2.0 ** -8   # half a step of bfloat16


def close(got, want, times=1.0, least=2.0 ** -20):
    """within `times` roundings to bfloat16, of values that were both rounded, and `least` of the largest"""
    got, want = got.double(), want.double()
    return bool(((got - want).abs() <= 2 * times * EPS * want.abs() + least * want.abs().max()).all())


def test_norm_of_more_elements_than_32_bits(handle):
    import torch
    import mluop_hip
    room_for(40)
    rows, channels, some = (1 << 22) + 1027, 512, 1500
    assert rows * channels > 2 ** 31
    g = torch.Generator(device="cuda").manual_seed(1)
    w, b = 1 + 0.2 * torch.randn(channels, device="cuda", generator=g), torch.randn(channels, device="cuda", generator=g)
    x = torch.randn(rows, channels, device="cuda", generator=g, dtype=torch.bfloat16)
    out, mean, rstd = mluop_hip.layer_norm_forward(handle, x, w, b)
    for at in (slice(0, some), slice(rows - some, rows)):
        want = torch.nn.functional.layer_norm(x[at].double(), (channels,), w.double(), b.double(), 1e-5)
        assert close(out[at], want)
    # a gradient of ones: every channel of the bias has as many as there are rows, which fp32 holds
    dx, dw, db = mluop_hip.layer_norm_backward(handle, torch.ones_like(x), x, w, b, mean, rstd)
    assert bool((db == rows).all())
    for at in (slice(0, some), slice(rows - some, rows)):
        leaf = x[at].double().requires_grad_()
        want = torch.autograd.grad(torch.nn.functional.layer_norm(leaf, (channels,), w.double(), b.double(), 1e-5).sum(), leaf)[0]
        # (w less its mean, and less its share along the row: sums of 512 products of fp32 with errors of 2^-24 each)
        assert close(dx[at], want, least=2.0 ** -13)
    total = torch.zeros(channels, device="cuda", dtype=torch.float64)
    for first in range(0, rows, 1 << 18):
        at = slice(first, min(first + (1 << 18), rows))
        # (a product with ones: torch's sums of many rows by several workgroups have been off)
        terms = ((x[at].float() - mean[at, None]) * rstd[at, None]).double()
        total += (torch.ones(1, terms.shape[0], device="cuda", dtype=torch.float64) @ terms)[0]
    # (a sum of 2^22 numbers of about one, some 2^11 of them one after the other: its size stays below 2^14 or so, and 2^12
    # roundings of half a step of that are 4)
    assert bool(((dw.double() - total).abs() <= 4.0).all())


def test_recurrence_of_more_elements_than_32_bits(handle):
    """gates of zero halve what was: 64 rows away nothing of it is left"""
    import torch
    import mluop_hip
    room_for(60)
    rows, channels, some, far = (1 << 21) + 777, 1024, 700, 64
    assert rows * channels > 2 ** 31
    g = torch.Generator(device="cuda").manual_seed(2)
    x = torch.randn(rows, channels, device="cuda", generator=g, dtype=torch.bfloat16)
    gates, dh = torch.zeros_like(x), torch.randn(rows, channels, device="cuda", generator=g, dtype=torch.bfloat16)
    for reverse in (False, True):
        out, final, carries = mluop_hip.gated_scan_forward(handle, x, gates, reverse=reverse)
        dx, dg, _ = mluop_hip.gated_scan_backward(handle, dh, None, x, gates, carries, reverse=reverse)
        for at in (slice(0, some), slice(rows - some, rows)):
            part = [t[at].contiguous() for t in (x, gates, dh)]
            o, f, c = mluop_hip.gated_scan_forward(handle, part[0], part[1], reverse=reverse)
            px, pg, _ = mluop_hip.gated_scan_backward(handle, part[2], None, part[0], part[1], c, reverse=reverse)
            inner = slice(far, some - far)
            for whole, piece in ((out, o), (dx, px), (dg, pg)):
                assert close(whole[at][inner], piece[inner])
        last = out[0] if reverse else out[-1]
        assert close(final[0], last)
        del out, carries, dx, dg


def test_recurrence_of_very_many_samples(handle):
    """more samples, and more tiles, than a grid has workgroups along y; most samples are empty and hand their states on"""
    import torch
    import mluop_hip
    rows, samples, channels = 300_000, 400_001, 64
    g = torch.Generator(device="cuda").manual_seed(3)
    x, gates, dh = (torch.randn(rows, channels, device="cuda", generator=g) for _ in range(3))
    initial, df = (torch.randn(samples, channels, device="cuda", generator=g) for _ in range(2))
    cuts = torch.randint(0, rows // 4, (samples - 1,), device="cuda", generator=g).sort().values * 4
    starts = torch.cat([torch.zeros_like(cuts[:1]), cuts, torch.full_like(cuts[:1], rows)]).to(torch.int32)
    filled = starts[1:] > starts[:-1]
    # (4096 rows and fewer have other ways)
    assert int(filled.sum()) > 1000 and int((~filled).sum()) > 70_000
    own = torch.cat([starts[:-1][filled], starts[-1:]])
    for reverse in (False, True):
        out, final, carries = mluop_hip.gated_scan_forward(handle, x, gates, starts, initial, reverse=reverse)
        ref, ref_final, ref_carries = mluop_hip.gated_scan_forward(handle, x, gates, own, initial[filled], reverse=reverse)
        assert torch.equal(out, ref) and torch.equal(final[filled], ref_final) and torch.equal(final[~filled], initial[~filled])
        got = mluop_hip.gated_scan_backward(handle, dh, df, x, gates, carries, starts, reverse=reverse)
        want = mluop_hip.gated_scan_backward(handle, dh, df[filled], x, gates, ref_carries, own, reverse=reverse)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        assert torch.equal(got[2][filled], want[2]) and torch.equal(got[2][~filled], df[~filled])


def test_rows_by_expert_of_more_elements_than_32_bits(handle):
    import torch
    import mluop_hip
    room_for(60)
    rows, choices, experts, channels = 1_100_003, 2, 8, 1024
    assert rows * choices * channels > 2 ** 31
    g = torch.Generator(device="cuda").manual_seed(4)
    first = torch.randint(0, experts, (rows, 1), device="cuda", generator=g)
    chosen = torch.cat([first, (first + 3) % experts], 1)
    chosen[::1000, 1] = -1
    x = torch.randn(rows, channels, device="cuda", generator=g, dtype=torch.bfloat16)
    ordered, starts, places = mluop_hip.expert_order(handle, chosen, experts)
    flat = torch.where(chosen < 0, experts, chosen).reshape(-1)
    by = torch.sort(flat, stable=True).indices
    sent = int(starts[-1])
    assert sent == int((chosen >= 0).sum()) and torch.equal(ordered[:sent].long(), by[:sent] // choices)
    assert bool((ordered[sent:] == -1).all()) and bool((places[::1000, 1] == -1).all())
    to = mluop_hip.expert_dispatch(handle, x, places, starts)
    for at in (slice(0, 1000), slice(sent - 1000, sent)):
        assert torch.equal(to[at], x[ordered[at].long()])
    assert not bool(to[sent:].any())
    back = mluop_hip.expert_combine(handle, to, places)
    twice = torch.where((chosen >= 0).all(1)[:, None], 2.0, 1.0).bfloat16()
    assert torch.equal(back[:1000], x[:1000] * twice[:1000]) and torch.equal(back[-1000:], x[-1000:] * twice[-1000:])
    weights = torch.full((rows, choices), 0.5, device="cuda")
    dy, dw = mluop_hip.expert_combine_backward(handle, x, to, places, weights, starts)
    for at in (slice(0, 1000), slice(sent - 1000, sent)):
        assert torch.equal(dy[at], x[ordered[at].long()] * 0.5)
    assert not bool(dy[sent:].any())
    for at in (slice(0, 1000), slice(rows - 1000, rows)):
        # (1024 squares in 32 bits)
        want = x[at].double().square().sum(1)[:, None].expand(-1, 2)
        want = torch.where(chosen[at] >= 0, want, torch.zeros_like(want))
        assert bool(((dw[at].double() - want).abs() <= 2.0 ** -14 * want).all())


@pytest.mark.parametrize("index", ["int32", "int64"])
def test_order_of_many_choices(handle, index):
    import torch
    import mluop_hip
    room_for(4)
    n, experts = 20_000_003, 2047
    g = torch.Generator(device="cuda").manual_seed(5)
    chosen = torch.randint(-2, experts + 2, (n, 1), device="cuda", generator=g).to(getattr(torch, index))
    ordered, starts, places = mluop_hip.expert_order(handle, chosen, experts)
    flat = torch.where((chosen >= 0) & (chosen < experts), chosen, experts).reshape(-1)
    by, rows = torch.sort(flat, stable=True)
    assert torch.equal(starts.long(), torch.searchsorted(by, torch.arange(experts + 1, device="cuda").to(by.dtype)))
    sent = int(starts[-1])
    assert torch.equal(ordered[:sent].long(), rows[:sent]) and bool((ordered[sent:] == -1).all())
    assert torch.equal(places[:, 0] >= 0, flat < experts)
    assert torch.equal(ordered[places[:, 0][flat < experts].long()].long(), torch.arange(n, device="cuda")[flat < experts])


def test_dropout_of_more_elements_than_32_bits(handle):
    """counters go on behind the element 2^32, and the number of the call has 64 bits"""
    import numpy as np
    import torch
    import mluop_hip
    from philox_reference import LOW, SHIFT, words
    room_for(40)
    n, p, seed, call = (1 << 32) + 8 * 5000 + 3, 0.25, 77, (1 << 33) + 5
    state = torch.tensor([seed, call], device="cuda")
    x = torch.ones(n, device="cuda", dtype=torch.bfloat16)
    out = mluop_hip.dropout_add_forward(handle, x, None, p, state)
    for first in (0, (1 << 32) - 8 * 4000, (n - 8 * 4000) // 8 * 8):
        some = min(8 * 4000, n - first)
        group = np.arange(first // 8, -(-(first + some) // 8), dtype=np.uint64)
        of_call = [np.full_like(group, call & 0xFFFFFFFF), np.full_like(group, call >> 32)]
        counter = np.stack([group & LOW, group >> SHIFT] + of_call, -1)
        w = words(counter, (seed, 0))
        halves = np.stack([w & np.uint32(0xFFFF), w >> np.uint32(16)], -1).reshape(-1)[:some]
        want = torch.from_numpy(halves >= 16384).cuda() * (65536 / 49152)
        assert torch.equal(out[first:first + some], want.bfloat16())


def jobs():
    """programs of the four operators, forward and backward, each on tensors of its own"""
    import torch
    from mluop_hip import nn as spnn

    def make(seed):
        g = torch.Generator(device="cuda").manual_seed(seed)
        rows, channels = 700 + 900 * seed, 64 + 32 * (seed % 3)
        x, gates, r = (torch.randn(rows, channels, device="cuda", generator=g) for _ in range(3))
        weight, bias = (torch.randn(channels, device="cuda", generator=g) for _ in range(2))
        starts = torch.tensor([0, rows // 3, rows], dtype=torch.int32, device="cuda")
        chosen = torch.randint(-1, 6, (rows, 2), device="cuda", generator=g)
        share, state = torch.rand(rows, 2, device="cuda", generator=g), torch.tensor([seed, 1], device="cuda")

        def run():
            leaves = [t.clone().requires_grad_() for t in (x, gates, weight, bias, share)]
            y = spnn.layer_norm(leaves[0], leaves[2], leaves[3])
            y, final = spnn.gated_scan(y, leaves[1], starts, reverse=seed % 2 == 1)
            _, first, places = spnn.expert_order(chosen, 6)
            y = spnn.expert_combine(spnn.expert_dispatch(y, places, first), places, first, leaves[4])
            y = spnn.dropout_add(y, r, 0.2, state)
            return [y.detach(), final.detach()] + list(torch.autograd.grad(y.square().sum() + final.sum(), leaves))
        return run
    return [make(s) for s in range(5)]


@pytest.mark.parametrize("streams", [False, True])
def test_several_threads(streams):
    """on one stream, whose library handle they share, or on one each"""
    import torch
    import mluop_hip
    guard, mluop_hip.GUARD_BYTES = mluop_hip.GUARD_BYTES, 0
    try:
        todo = jobs()
        alone = [job() for job in todo]
        torch.cuda.synchronize()
        problems, gate = [], threading.Barrier(len(todo))

        def work(n):
            try:
                gate.wait(60)
                stream = torch.cuda.Stream() if streams else torch.cuda.current_stream()
                with torch.cuda.stream(stream):
                    for r in range(6):
                        got = todo[n]()
                        stream.synchronize()
                        for i, (a, b) in enumerate(zip(got, alone[n])):
                            if not torch.equal(a, b):
                                problems.append("thread %d, round %d: output %d differs" % (n, r, i))
            except Exception as e:  # noqa: BLE001 (reported by the main thread)
                problems.append("thread %d: %r" % (n, e))
        pool = [threading.Thread(target=work, args=(n,)) for n in range(len(todo))]
        for t in pool:
            t.start()
        for t in pool:
            t.join(100)
        assert not any(t.is_alive() for t in pool)
        torch.cuda.synchronize()
        assert not problems, problems[:5]
    finally:
        mluop_hip.GUARD_BYTES = guard


def test_several_streams_of_one_thread():
    """enqueued one behind the other without a wait: workspaces of one call are not another's"""
    import torch
    import mluop_hip
    guard, mluop_hip.GUARD_BYTES = mluop_hip.GUARD_BYTES, 0
    try:
        todo = jobs()
        alone = [job() for job in todo]
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream() for _ in todo]
        for _ in range(4):
            found = []
            for job, stream in zip(todo, streams):
                with torch.cuda.stream(stream):
                    found.append(job())
            torch.cuda.synchronize()
            for got, want in zip(found, alone):
                assert all(torch.equal(a, b) for a, b in zip(got, want))
    finally:
        mluop_hip.GUARD_BYTES = guard


@pytest.mark.parametrize("share", [0.03, 0.6, 1.0])
def test_very_many_choices_of_no_expert(gpu_handle, share):
    """their places are zero, in the order and in the gradients of a weighted sum"""
    import torch
    import mluop_hip
    rows, choices, channels = 30_001, 3, 72
    g = torch.Generator(device="cuda").manual_seed(int(100 * share))
    chosen = torch.randint(0, 9, (rows, choices), device="cuda", generator=g)
    chosen[torch.rand((rows, choices), device="cuda", generator=g) < share] = -1
    x = torch.randn(rows, channels, device="cuda", generator=g).half()
    ordered, starts, places = mluop_hip.expert_order(gpu_handle, chosen, 9)
    sent = int(starts[-1])
    assert sent == int((chosen >= 0).sum())
    to = mluop_hip.expert_dispatch(gpu_handle, x, places, starts)
    assert torch.equal(to[:sent], x[ordered[:sent].long()]) and not bool(to[sent:].any())
    w = torch.rand(rows, choices, device="cuda", generator=g)
    dy, dw = mluop_hip.expert_combine_backward(gpu_handle, x, to, places, w, starts)
    assert not bool(dy[sent:].any()) and bool((dw[chosen < 0] == 0).all())
    there = places >= 0
    want = (x.float().unsqueeze(1) * w.unsqueeze(2))[there].half()
    assert torch.equal(dy[places[there].long()], want)


@pytest.mark.parametrize("starts", [[0, 1000, 100_000], [200_000, 200_000, 299_000], [7, 7]])
def test_very_many_rows_of_no_sample(gpu_handle, starts):
    """rows in front of the first sample and behind the last are zero in every result, whatever they hold"""
    import torch
    import mluop_hip
    rows, channels = 300_001, 48
    g = torch.Generator(device="cuda").manual_seed(6)
    x, gates, dh = (torch.randn(rows, channels, device="cuda", generator=g).bfloat16() for _ in range(3))
    for t in (x, gates, dh):
        t[:starts[0]] = float("nan")
        t[starts[-1]:] = float("nan")
    where = torch.tensor(starts, dtype=torch.int32, device="cuda")
    out, final, carries = mluop_hip.gated_scan_forward(gpu_handle, x, gates, where)
    dx, dg, _ = mluop_hip.gated_scan_backward(gpu_handle, dh, None, x, gates, carries, where)
    for t in (out, dx, dg):
        assert not bool(t[:starts[0]].any()) and not bool(t[starts[-1]:].any()) and not bool(t.isnan().any())
    assert not bool(final.isnan().any())
