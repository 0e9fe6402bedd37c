"""The gated recurrence over samples of so many tiles that they are joined in several turns of 1024: memories that last across all
of them, with counts of states around a turn's and two turns', for every length of a tile."""
import pytest

pytestmark = pytest.mark.gpu

TURN = 1024   # states in front of tiles that are worked out together


def sizes(tile):
    """rows of samples with one turn's states but one, as many, one more, and one more than two turns'"""
    return [TURN * tile, TURN * tile + 1, (TURN + 1) * tile + tile // 2, (2 * TURN + 1) * tile + 5]


def long_memories(rows, channels, samples, tile, kind):
    """Numbers of one sign, so that no state's parts cancel; decays of which a turn's tiles leave some e^-1.5; and states in front
    and behind of 20 times what the recurrence comes to, so that a state which is missing, or is that of the turn before, is off by
    several times the bound, which adds up some 10 units of 2^-24 for every row."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(rows + channels)

    def rand(*shape):
        return torch.rand(*shape, device="cuda", generator=g) + 0.5
    rest = rand(rows, channels) * (1.5 / (TURN * tile))   # 1 - a
    gates = torch.log((1 - rest) / rest) if kind == "sigmoid" else -rest
    reach = TURN * tile / 1.5   # rows that a sum without weights reaches
    h0, df = 20 * (1.0 if kind == "sigmoid" else reach) * rand(samples, channels), 20 * reach * rand(samples, channels)
    return rand(rows, channels), gates, h0, rand(rows, channels), df


@pytest.mark.parametrize("channels,tile,samples", [(40, 64, 4), (16, 128, 1), (8, 256, 1)])
@pytest.mark.parametrize("kind,reverse", [("sigmoid", False), ("exp", True)])
def test_samples_of_several_turns(gpu_handle, channels, tile, samples, kind, reverse):
    from test_gpu_gated_scan import check
    rows = sizes(tile) if samples == 4 else [(TURN + 1) * tile + tile // 2]
    print("gated scan in turns", channels, rows, kind, reverse, flush=True)
    starts = [sum(rows[:k]) for k in range(samples + 1)]
    x, g, h0, dh, df = long_memories(starts[-1], channels, samples, tile, kind)
    check(gpu_handle, x, g, starts, h0, dh, df, kind, reverse, "float32")
