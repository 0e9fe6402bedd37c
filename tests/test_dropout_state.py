"""The seed and the count of a DropoutAdd: modules made on the meta device and loaded, modules that begin anew, deep copies."""
import copy

import pytest


def counting(monkeypatch):
    """the states of the calls, without a GPU"""
    from mluop_hip import nn as spnn
    seen = []

    def call(features, residual, p, state):
        seen.append(state.tolist())
        return features
    monkeypatch.setattr(spnn, "dropout_add", call)
    return seen


@pytest.mark.parametrize("seed", [None, 5])
def test_made_without_memory_and_loaded(monkeypatch, seed):
    import torch
    from mluop_hip import nn as spnn
    seen = counting(monkeypatch)
    with torch.device("meta"):
        layer = spnn.DropoutAdd(0.5, seed=seed)
    assert layer.state.is_meta
    layer.to_empty(device="cpu")
    # (whatever the memory held)
    for buffer in layer.buffers():
        buffer.fill_(77)
    layer.load_state_dict({"state": torch.tensor([11, 4])})
    for _ in range(3):
        layer(torch.zeros(2))
    assert seen == [[11, 4], [11, 5], [11, 6]] and layer.state.tolist() == [11, 7]


def test_made_without_memory_and_begun_anew():
    import torch
    from mluop_hip import nn as spnn
    with torch.device("meta"):
        given, drawn = spnn.DropoutAdd(0.5, seed=5), spnn.DropoutAdd(0.5)
    for layer in (given, drawn):
        layer.to_empty(device="cpu")
        layer.state.fill_(-1)
        layer.reset_parameters()
    assert given.state.tolist() == [5, 0]
    assert 0 <= int(drawn.state[0]) < 2 ** 62 and int(drawn.state[1]) == 0


def test_only_the_state_is_kept():
    from mluop_hip import nn as spnn
    layer = spnn.DropoutAdd(0.5, seed=5)
    assert list(layer.state_dict()) == ["state"] and [n for n, _ in layer.named_buffers()] == ["state"]


def test_deep_copies_go_on_as_their_original_until_they_begin_anew(monkeypatch):
    import torch
    from mluop_hip import nn as spnn
    seen = counting(monkeypatch)
    torch.manual_seed(3)
    layer = spnn.DropoutAdd(0.5)
    layer(torch.zeros(2))
    twin = copy.deepcopy(layer)
    layer(torch.zeros(2))
    twin(torch.zeros(2))
    assert seen[1] == seen[2] and seen[1][1] == 1
    twin.reset_parameters()
    assert int(twin.state[0]) != int(layer.state[0]) and int(twin.state[1]) == 0
    torch.manual_seed(3)
    assert int(spnn.DropoutAdd(0.5).state[0]) == seen[0][0]
