"""Trains a small network over labelled voxels with the operators around the sparse convolutions: learned rows for the
voxels' categories, submanifold convolutions with group norm and SiLU between them, a layer of experts on every voxel, and the
AdamW step with 8-bit states.

    python examples/voxel_experts.py [--steps 60] [--rows 20000] [--dtype bfloat16]

Synthetic clouds: a voxel's category is drawn at random, its label is the commonest category parity around it, which a
network can only tell from the neighbours."""
import argparse
import os
import sys

import numpy as np
import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "mlu-ops_amd", "python"))
from mluop_hip import datagen, nn as spnn, optim  # noqa: E402

CATEGORIES, CHANNELS, CLASSES, BATCH = 40, 64, 2, 2
SPACE = (16, 96, 96)


class Net(torch.nn.Module):
    def __init__(self):
        super().__init__()
        self.embed = spnn.Embedding(CATEGORIES, CHANNELS, scale=1.0)
        self.encoder = spnn.SparseSequential(
            spnn.SubMConv3d(CHANNELS, CHANNELS, 3, indice_key="cells"), spnn.GroupNormAct(16, CHANNELS, activation="silu"),
            spnn.SubMConv3d(CHANNELS, CHANNELS, 3, indice_key="cells"), spnn.GroupNormAct(16, CHANNELS, activation="silu"))
        self.experts = spnn.ExpertMLP(CHANNELS, 2 * CHANNELS, experts=8, choices=2)
        self.head = torch.nn.Linear(CHANNELS, CLASSES)

    def forward(self, categories, indices, dtype):
        x = spnn.SparseTensor(self.embed(categories).to(dtype), indices, SPACE, BATCH, distinct=True, ordered=True)
        features = self.encoder(x).features
        features = features + self.experts(features)
        return self.head(features.float())


def cloud(rows, seed):
    """(categories [rows], indices [rows, 4] in cell order, labels [rows]) on the GPU"""
    g = torch.Generator(device="cuda").manual_seed(seed)
    idx = datagen.clustered_voxels((BATCH,) + SPACE, rows // BATCH, seed)
    linear = ((idx[:, 0].astype(np.int64) * SPACE[0] + idx[:, 1]) * SPACE[1] + idx[:, 2]) * SPACE[2] + idx[:, 3]
    indices = torch.from_numpy(np.ascontiguousarray(idx[np.argsort(linear)], dtype=np.int32)).cuda()
    categories = torch.randint(0, CATEGORIES, (indices.shape[0],), device="cuda", generator=g, dtype=torch.int32)
    odd = torch.zeros((BATCH,) + tuple(s + 2 for s in SPACE), device="cuda")
    n, d, h, w = indices.long().unbind(1)
    odd[n, d + 1, h + 1, w + 1] = torch.where(categories % 2 == 1, 1.0, -1.0)
    around = torch.nn.functional.conv3d(odd[:, None], torch.ones(1, 1, 3, 3, 3, device="cuda"))[:, 0]
    return categories, indices, (around[n, d, h, w] > 0).long()


def train(steps, rows, dtype, report=None):
    torch.manual_seed(0)
    net = Net().cuda()
    step = optim.AdamW(net.parameters(), lr=3e-3, weight_decay=0.01, state_bits=8)
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
