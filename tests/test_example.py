"""The example that runs the stream embedding and the 8-bit checkpoints together."""
import importlib.util
import os

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def load():
    spec = importlib.util.spec_from_file_location("train_streams", os.path.join(ROOT, "examples", "train_streams.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


def test_example_names_public_operators():
    m = load()
    model = m.Model(vocab=50, hidden=32, blocks=1)
    assert model.embed.weight.shape == (50, 32) and model.blocks[0].mix.checkpoint_8bit
    assert not model.embed.weight[0].any()


@pytest.mark.gpu
def test_example_trains_like_full_precision_and_keeps_less(cuda):
    m = load()
    eight, kept8 = m.train(steps=12)
    full, kept = m.train(steps=12, eight=False)
    assert eight[0] == pytest.approx(full[0], rel=1e-5)  # the forward passes are the same formulas in fp32
    assert eight[-1] < 0.7 * eight[0] and full[-1] < 0.7 * full[0]
    # gradients differ by 8-bit rounding of the activations (about 0.6% of their size), averaged over 512 tokens
    assert abs(eight[-1] - full[-1]) < 0.05 * full[0]
    assert kept8 < 0.6 * kept


@pytest.mark.gpu
def test_a_step_is_reproducible(cuda):
    """The operators' own parts: two backward passes give the same bits."""
    m = load()
    torch.manual_seed(1)
    model = m.Model(vocab=100, hidden=64, blocks=1).to(cuda)
    ids = torch.randint(1, 100, (4, 33), device=cuda)
    grads = []
    for _ in range(2):
        model.zero_grad()
        h = model.embed(ids.reshape(-1))
        model.blocks[0].mix(h).square().sum().backward()
        grads.append([p.grad.clone() for p in (model.embed.weight, *model.blocks[0].mix.parameters())])
    assert all(torch.equal(a, b) for a, b in zip(*grads))
