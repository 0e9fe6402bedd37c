"""The gated recurrence's decays by themselves: samples of one row from a state of one, or with features of one, give a and 1 - a
as the kernels have them, over the whole range of gates.

In units of 2^-24 of the result: the exponential e of the kernels is off by 2 for that of a power of two and by 1 for the step
that puts the power right, 3; a sum, a difference or a product is off by 1, a reciprocal by 2.
  1 - a = 1 / (1 + e)      of e its share e / (1 + e), 1 for the sum, 2: at most 6
  a = e / (1 + e), g < 0   of e its share 1 / (1 + e), 1, 2, and 1 for the product: at most 7
  a = 1 - 1 / (1 + e)      the reciprocal is at most a, and its 6 at most 6 of a, and 1: at most 7
Rows of 16 bits take the power of the rounded product p of g with log2(e), whose half step is |p| ln(2) = |g| units of e, and
whose constant is off by 0.23 units of itself, so of e by 0.23 |g|: 1.23 |g| in place of the step that puts it right."""
import pytest

pytestmark = pytest.mark.gpu

UNIT, LEAST = 2.0 ** -24, 2.0 ** -126
EXP, DECAY, REST = 3, 7, 6


def gates(most):
    """negative and positive ones, from tiny to `most`, in rows of 32"""
    import torch
    g = torch.Generator(device="cuda").manual_seed(0)
    spread = (torch.rand(2, 200_000, device="cuda", generator=g) * 2 - 1) * most
    small = torch.exp(-16 * torch.rand(2, 20_000, device="cuda", generator=g)) * torch.tensor([[1.0], [-1.0]], device="cuda")
    whole = torch.arange(-int(most), int(most) + 1, device="cuda", dtype=torch.float32)
    all_of_them = torch.cat([spread.view(-1), small.view(-1), whole, whole * 0.69314718, torch.zeros(32, device="cuda")])
    return all_of_them[:all_of_them.numel() // 32 * 32].view(-1, 32).contiguous()


def off(got, want, more=0.0):
    """units beyond what flushing the least numbers and `more` units explain"""
    room = ((got.double() - want).abs() - LEAST - more * UNIT * want).clamp(min=0)
    return float((room / want).max()) / UNIT


@pytest.mark.parametrize("kind,most", [("sigmoid", 87.0), ("exp", 87.0)])
@pytest.mark.parametrize("way", ["whole", "joined"])
def test_units(gpu_handle, kind, most, way):
    """whole: samples of one row, some thousands of them at a time; joined: more rows than that, by other kernels"""
    import torch
    import mluop_hip
    print("decays", kind, way, flush=True)
    g = gates(most)
    if way == "whole":
        g = g[:2000]
    rows, channels = g.shape
    starts = torch.arange(rows + 1, dtype=torch.int32, device="cuda")
    zero, one = torch.zeros_like(g), torch.ones_like(g)
    wide = g.double()
    a = torch.exp(wide) if kind == "exp" else 1.0 / (1.0 + torch.exp(-wide))
    u = torch.ones_like(wide) if kind == "exp" else 1.0 / (1.0 + torch.exp(wide))
    of_a = EXP if kind == "exp" else DECAY
    out, final, carries = mluop_hip.gated_scan_forward(gpu_handle, zero, g, starts, one, kind)
    found = {"out": off(out, a), "final": off(final, a)}
    assert max(found.values()) <= of_a, found
    # dx = u, initial's a, and the gate's a u (1 - 0) or a: a product or two more
    dx, dg, di = mluop_hip.gated_scan_backward(gpu_handle, one, None, zero, g, carries, starts, kind)
    found = {"features_grad": off(dx, u) / (REST if kind == "sigmoid" else 1), "initial_grad": off(di, a) / of_a,
             "gates_grad": off(dg, a * u) / (of_a + (REST + 1 if kind == "sigmoid" else 0))}
    assert max(found.values()) <= 1, found
    if kind == "sigmoid":
        out, final, _ = mluop_hip.gated_scan_forward(gpu_handle, one, g, starts, None, kind)
        found = {"out": off(out, u), "final": off(final, u)}
        assert max(found.values()) <= REST, found


def test_values_that_are_exact(gpu_handle):
    """no change at a gate of zero with exp, or where an exponential is zero or infinite; a gate that is no number gives none"""
    import torch
    import mluop_hip
    inf, nan = float("inf"), float("nan")
    g = torch.tensor([[0.0, -inf, -1e30, -200.0, inf, 1e30, 200.0, nan]], device="cuda")
    one, zero = torch.ones_like(g), torch.zeros_like(g)

    def decay(kind):
        return mluop_hip.gated_scan_forward(gpu_handle, zero, g, None, one, kind)[0][0].tolist()
    got = decay("exp")
    assert got[:7] == [1.0, 0.0, 0.0, 0.0, inf, inf, inf] and got[7] != got[7]
    got = decay("sigmoid")
    assert got[:7] == [0.5, 0.0, 0.0, 0.0, 1.0, 1.0, 1.0] and got[7] != got[7]


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("kind", ["sigmoid", "exp"])
def test_states_of_16_bit_rows(gpu_handle, dtype, kind):
    """the states behind samples of one row, and the gradients of those in front, are fp32"""
    import torch
    import mluop_hip
    g = gates(87.0).to(getattr(torch, dtype))
    starts = torch.arange(g.shape[0] + 1, dtype=torch.int32, device="cuda")
    zero, one = torch.zeros_like(g), torch.ones(g.shape, device="cuda")
    wide = g.double()
    a = torch.exp(wide) if kind == "exp" else 1.0 / (1.0 + torch.exp(-wide))
    of_a, more = (EXP if kind == "exp" else DECAY), 1.23 * wide.abs()
    _, final, carries = mluop_hip.gated_scan_forward(gpu_handle, zero, g, starts, one, kind)
    _, _, di = mluop_hip.gated_scan_backward(gpu_handle, zero, one, zero, g, carries, starts, kind)
    found = {"final": off(final, a, more), "initial_grad": off(di, a, more)}
    assert max(found.values()) <= of_a, found
