"""Dropout layers in a model: which numbers each draws, what a second run draws, and what
data-parallel wrapping and checkpoints do to them."""
import copy
import os
import pickle
import socket

import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp
from torch import nn
from torch.utils.checkpoint import checkpoint

import mhc_ascend_b200 as mhc


def seeds(module):
    return [m.state[0].item() for m in module.modules() if isinstance(m, mhc.DropoutCounter)]


# ---------------------------------------------------------------------------
# no GPU needed: layers without a seed
# ---------------------------------------------------------------------------

def test_layers_without_a_seed_differ():
    model = nn.ModuleList([mhc.StreamDropout(0.1) for _ in range(5)] +
                          [mhc.MHCResidualWrapper(8, 4, branch_dropout=0.1) for _ in range(5)])
    assert len(set(seeds(model))) == 10
    assert seeds(mhc.StreamDropout(0.1, seed=7)) == [7] and seeds(mhc.MHCResidualWrapper(8, branch_dropout=0.1, dropout_seed=7)) == [7]
    state = torch.random.get_rng_state()
    mhc.StreamDropout(0.1)
    assert torch.equal(torch.random.get_rng_state(), state)  # the parameters' initial values stay what they are


def test_copies_of_layers():
    """A block copied for each layer of a model; a saved or pickled layer goes on as it was."""
    block = nn.Sequential(nn.Linear(4, 4), mhc.StreamDropout(0.1), mhc.MHCResidualWrapper(8, branch_dropout=0.2))
    model = nn.ModuleList(copy.deepcopy(block) for _ in range(4))
    assert len(set(seeds(model) + seeds(block))) == 10
    assert all(torch.equal(b[0].weight, block[0].weight) and b[1].p == 0.1 for b in model)
    given = mhc.StreamDropout(0.1, seed=3)
    assert seeds(copy.deepcopy(given)) == [3]  # as asked for
    assert seeds(pickle.loads(pickle.dumps(block))) == seeds(block)
    model[0].load_state_dict(block.state_dict())
    assert seeds(model[0]) == seeds(block)
    shared = copy.deepcopy(nn.ModuleList([block[1], block[1]]))
    assert shared[0] is shared[1]
    frozen = copy.deepcopy(block).requires_grad_(False).eval()
    assert frozen[1](torch.ones(2)).tolist() == [1, 1]


@pytest.mark.gpu
def test_layers_without_a_seed_drop_other_places(cuda):
    model = nn.ModuleList(mhc.StreamDropout(0.5) for _ in range(4)).to(cuda)
    model.append(copy.deepcopy(model[0]))
    x = torch.ones(4096, device=cuda)
    masks = [layer(x) != 0 for layer in model]
    for i in range(5):
        for j in range(i):  # 4096 coins each: half of them meet, give or take 6 deviations
            assert abs((masks[i] == masks[j]).float().mean().item() - 0.5) < 6 * 0.5 / 64
