"""A small mHC language model whose activations are kept in 8 bits.

Token ids become n residual streams (``StreamEmbedding``); each block mixes the
streams (``MHCLayer``, streams kept in 8 bits) and adds a feed-forward branch
whose norm and linear layers keep their inputs in 8 bits; the streams' mean is
normalised and projected to the vocabulary, and the loss is the tokens' negative
log probability (``token_logprobs``).  Trains on one random batch:

    python examples/train_streams.py [--full] [--steps 30] [--dropout 0.1]

``--full`` keeps the activations in full precision for comparison, ``--dropout``
drops branch outputs out; the script prints the loss, what the activations of a
step take, and the most likely next tokens of the first text.
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
    def __init__(self, hidden, n, eight, dropout=0.0, seed=0):
        super().__init__()
        self.eight = eight
        self.dropout = mhc.StreamDropout(dropout, seed)
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
        return x + self.dropout(h).unsqueeze(1)


class Model(nn.Module):
    def __init__(self, vocab=1000, hidden=256, n=4, blocks=2, eight=True, dropout=0.0):
        super().__init__()
        self.embed = mhc.StreamEmbedding(vocab, hidden, n, scale=[1.0, 0.5, 0.25, 0.125][:n], padding_idx=0)
        self.blocks = nn.ModuleList(Block(hidden, n, eight, dropout, seed=i) for i in range(blocks))
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


def loss_of(logits, targets):
    """Mean negative log probability of the targets; token 0 is padding."""
    logprob = mhc.token_logprobs(logits, targets, ignore_index=0).logprob
    return -logprob.sum() / (targets != 0).sum()


def train(steps=30, batch=8, length=64, vocab=1000, eight=True, dropout=0.0, device="cuda", answer=False):
    """Losses of `steps` steps on one batch, and the bytes that a step's
    activations take; with `answer` also the five most likely next tokens at each
    place of the first text, and their log probabilities."""
    torch.manual_seed(0)
    model = Model(vocab, eight=eight, dropout=dropout).to(device)
    ids = torch.randint(1, vocab, (batch, length + 1), device=device)
    ids[:, -8:] = 0  # padding at the end
    opt = torch.optim.Adam(model.parameters(), lr=3e-3)
    losses, kept = [], 0
    for _ in range(steps):
        opt.zero_grad()
        before = torch.cuda.memory_allocated(device)
        loss = loss_of(model(ids[:, :-1]), ids[:, 1:].reshape(-1))
        kept = torch.cuda.memory_allocated(device) - before
        loss.backward()
        opt.step()
        losses.append(loss.item())
    if not answer:
        return losses, kept
    with torch.no_grad():
        best = mhc.token_logprobs(model.eval()(ids[:1, :-1]), ids[0, 1:], top=5)
    return losses, kept, best.top_id, best.top_logprob


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--steps", type=int, default=30)
    ap.add_argument("--full", action="store_true")
    ap.add_argument("--dropout", type=float, default=0.0)
    a = ap.parse_args()
    losses, kept, ids, logprobs = train(a.steps, eight=not a.full, dropout=a.dropout, answer=True)
    for i in range(0, len(losses), 5):
        print(f"step {i:3d}  loss {losses[i]:.4f}")
    print(f"last loss {losses[-1]:.4f}; activations of a step: {kept / 2 ** 20:.1f} MiB")
    for place in range(3):
        likely = ", ".join(f"{i} ({p:.2f})" for i, p in zip(ids[place].tolist(), logprobs[place].exp().tolist()))
        print(f"after token {place}: {likely}")
