"""Trains a small network that reads the voxels of a cloud one after the other: learned rows for their categories, then blocks of
layer norm, a gated recurrence forwards and one backwards, experts on every voxel, and residuals with dropout between them.

    python examples/voxel_sequence.py [--steps 60] [--rows 20000] [--dtype bfloat16]

Synthetic clouds: categories are drawn at random, and a voxel's label says which of two marking categories came last in its cloud,
which a network can only tell from all voxels in front."""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "mlu-ops_amd", "python"))
from mluop_hip import datagen, nn as spnn, optim  # noqa: E402

CATEGORIES, CHANNELS, CLASSES, BATCH = 40, 64, 2, 2
SPACE = (16, 96, 96)


class Mix(torch.nn.Module):
    """Rows of every sample mixed along their order, in both directions."""

    def __init__(self, channels, kind):
        super().__init__()
        self.forwards, self.backwards = (spnn.GatedScan(channels, kind=kind, reverse=r) for r in (False, True))

    def forward(self, x):
        return x.replace_features(self.forwards(x).features + self.backwards(x).features)


class Block(torch.nn.Module):
    def __init__(self, channels, kind="sigmoid", experts=8, dropout=0.1):
        super().__init__()
        self.norms = torch.nn.ModuleList([spnn.LayerNorm(channels) for _ in range(2)])
        self.mix = Mix(channels, kind)
        self.experts = spnn.ExpertMLP(channels, 2 * channels, experts, choices=2)
        self.residuals = torch.nn.ModuleList([spnn.DropoutAdd(dropout) for _ in range(2)])

    def forward(self, x):
        x = self.residuals[0](self.mix(self.norms[0](x)), x)
        normed = self.norms[1](x.features)
        return x.replace_features(self.residuals[1](self.experts(normed), x.features))


class Net(torch.nn.Module):
    def __init__(self):
        super().__init__()
        self.embed = spnn.Embedding(CATEGORIES, CHANNELS)
        self.blocks = torch.nn.Sequential(Block(CHANNELS, "sigmoid"), Block(CHANNELS, "exp"))
        self.norm, self.head = spnn.LayerNorm(CHANNELS), torch.nn.Linear(CHANNELS, CLASSES)

    def forward(self, categories, indices, dtype):
        x = spnn.SparseTensor(self.embed(categories).to(dtype), indices, SPACE, BATCH, distinct=True, ordered=True)
        return self.head(self.norm(self.blocks(x).features).float())


def cloud(rows, seed):
    """(categories [rows], indices [rows, 4] in cell order, labels [rows]) on the GPU"""
    g = torch.Generator(device="cuda").manual_seed(seed)
    indices = torch.from_numpy(datagen.clustered_voxels((BATCH,) + SPACE, rows // BATCH, seed)).cuda()
    categories = torch.randint(0, CATEGORIES, (indices.shape[0],), generator=g, device="cuda")
    # the place of the last marking category of each sample, in front of it or at a row
    place = torch.arange(indices.shape[0], device="cuda")
    marks = torch.where(categories < 2, place, torch.full_like(place, -1))
    last = torch.cummax(marks, dim=0).values
    starts = torch.searchsorted(indices[:, 0].contiguous(), indices[:, 0].contiguous())
    labels = torch.where(last >= starts, categories[last.clamp(min=0)], torch.zeros_like(categories))
    return categories, indices, labels


def train(steps, rows, dtype, seed=0, report=None):
    torch.manual_seed(seed)
    net = Net().cuda()
    step = optim.AdamW(net.parameters(), lr=3e-3, weight_decay=1e-3)
    losses = []
    for k in range(steps):
        categories, indices, labels = cloud(rows, k % 4)
        loss = torch.nn.functional.cross_entropy(net(categories, indices, dtype), labels)
        step.zero_grad()
        loss.backward()
        step.step()
        losses.append(loss.detach())
        if report is not None and (k + 1) % report == 0:
            print("step %d: loss %.4f" % (k + 1, float(losses[-1])), flush=True)
    return net, [float(v) for v in losses]


if __name__ == "__main__":
    parser = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    parser.add_argument("--steps", type=int, default=60)
    parser.add_argument("--rows", type=int, default=20_000)
    parser.add_argument("--dtype", default="bfloat16", choices=["float32", "float16", "bfloat16"])
    a = parser.parse_args()
    train(a.steps, a.rows, getattr(torch, a.dtype), report=10)
