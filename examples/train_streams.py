"""A small mHC language model whose activations are kept in 8 bits.

Token ids become n residual streams (``StreamEmbedding``); each block mixes the
streams (``MHCLayer``, streams kept in 8 bits) and adds a feed-forward branch
whose norm and linear layers keep their inputs in 8 bits; the streams' mean is
normalised and projected to the vocabulary.  Trains on one random batch:

    python examples/train_streams.py [--full] [--steps 30]

``--full`` keeps the activations in full precision for comparison; the script
prints the loss and what the activations of a step take.
"""
import argparse
import os
import sys

import torch
import torch.nn as nn
import torch.nn.functional as F

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import mhc_ascend_b200 as mhc  # noqa: E402
from mhc_ascend_b200.ops import stream_mean  # noqa: E402


class Block(nn.Module):
    def __init__(self, hidden, n, eight):
        super().__init__()
        self.eight = eight
        self.mix = mhc.MHCLayer(hidden, n, checkpoint_8bit=eight)
        self.norm = nn.Parameter(torch.ones(hidden))
        self.up = nn.Parameter(torch.randn(4 * hidden, hidden) * hidden ** -0.5)
        self.down = nn.Parameter(torch.randn(hidden, 4 * hidden) * (4 * hidden) ** -0.5)

    def forward(self, x):
        x = self.mix(x)
        h = stream_mean(x)
        if self.eight:
            h = mhc.linear_checkpoint8(mhc.rmsnorm_checkpoint8(h, self.norm), self.up)
            h = mhc.linear_checkpoint8(F.gelu(h), self.down)
        else:
            h = F.linear(F.gelu(F.linear(mhc.rmsnorm(h, self.norm), self.up)), self.down)
        return x + h.unsqueeze(1)


class Model(nn.Module):
    def __init__(self, vocab=1000, hidden=256, n=4, blocks=2, eight=True):
        super().__init__()
        self.embed = mhc.StreamEmbedding(vocab, hidden, n, scale=[1.0, 0.5, 0.25, 0.125][:n], padding_idx=0)
        self.blocks = nn.ModuleList(Block(hidden, n, eight) for _ in range(blocks))
        self.norm = nn.Parameter(torch.ones(hidden))
        self.head = nn.Parameter(torch.randn(vocab, hidden) * hidden ** -0.5)
        self.eight = eight

    def forward(self, ids):
        x = self.embed(ids.reshape(-1))
        for b in self.blocks:
            x = b(x)
        h = stream_mean(x)
        if self.eight:
            return mhc.linear_checkpoint8(mhc.rmsnorm_checkpoint8(h, self.norm), self.head)
        return F.linear(mhc.rmsnorm(h, self.norm), self.head)


def train(steps=30, batch=8, length=64, vocab=1000, eight=True, device="cuda"):
    """Losses of `steps` steps on one batch, and the bytes that a step's
    activations take."""
    torch.manual_seed(0)
    model = Model(vocab, eight=eight).to(device)
    ids = torch.randint(1, vocab, (batch, length + 1), device=device)
    ids[:, -8:] = 0  # padding at the end
    opt = torch.optim.Adam(model.parameters(), lr=3e-3)
    losses, kept = [], 0
    for _ in range(steps):
        opt.zero_grad()
        before = torch.cuda.memory_allocated(device)
        loss = F.cross_entropy(model(ids[:, :-1]), ids[:, 1:].reshape(-1), ignore_index=0)
        kept = torch.cuda.memory_allocated(device) - before
        loss.backward()
        opt.step()
        losses.append(loss.item())
    return losses, kept


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--steps", type=int, default=30)
    ap.add_argument("--full", action="store_true")
    a = ap.parse_args()
    losses, kept = train(a.steps, eight=not a.full)
    for i in range(0, len(losses), 5):
        print(f"step {i:3d}  loss {losses[i]:.4f}")
    print(f"last loss {losses[-1]:.4f}; activations of a step: {kept / 2 ** 20:.1f} MiB")
