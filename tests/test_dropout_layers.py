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


# ---------------------------------------------------------------------------
# a second run in the backward pass
# ---------------------------------------------------------------------------

class RunsAgain(torch.autograd.Function):
    """A function whose backward pass calls `again`, as a checkpoint's does."""

    @staticmethod
    def forward(ctx, x, again):
        ctx.again = again
        return x * 2

    @staticmethod
    def backward(ctx, grad):
        ctx.again()
        return grad * 2, None


def test_no_new_numbers_in_a_backward_pass():
    layer = mhc.StreamDropout(0.5, seed=1)
    x = torch.ones(4, requires_grad=True)
    for again in (lambda: layer.counter.take(4), lambda: layer(x), lambda: layer.take(x.shape)):
        with pytest.raises(RuntimeError, match="backward pass"):
            RunsAgain.apply(x, again).sum().backward()
    with pytest.raises(RuntimeError, match="CUDA"):  # and the numbers are free again
        layer.counter.take(4)
    RunsAgain.apply(x, lambda: layer.eval()(x)).sum().backward()  # the identity draws none


@pytest.mark.gpu
@pytest.mark.parametrize("reentrant", [True, False])
def test_torch_checkpoint_draws_no_other_mask(cuda, reentrant):
    layer = mhc.StreamDropout(0.4, seed=5).to(cuda)
    x = torch.randn(20, 64, device=cuda, requires_grad=True)
    out = checkpoint(lambda t: layer(t * t).sum(), x, use_reentrant=reentrant)
    with pytest.raises(RuntimeError, match="take them before"):
        out.backward()
    torch.cuda.synchronize()
    rng = layer.take(x.shape)
    out = checkpoint(lambda t: layer(t * t, rng), x, use_reentrant=reentrant)
    out.sum().backward()
    want = x.detach().clone().requires_grad_(True)
    same = layer(want * want, rng)
    same.sum().backward()
    assert torch.equal(out, same) and torch.equal(x.grad, want.grad)
    assert layer.counter.state.tolist() == [5, 2 * mhc.dropout_groups(x.shape)]  # of the first call and of take
    layer.eval()
    assert layer.take(x.shape) is None
    checkpoint(lambda t: layer(t * t, None), x, use_reentrant=reentrant).sum().backward()


@pytest.mark.gpu
@pytest.mark.parametrize("mode", ["fused", "kept", "packed"])
def test_wrapper_under_checkpoints(cuda, mode):
    """With numbers taken before, the same results and gradients as without a checkpoint."""
    n = 2 if mode == "packed" else 4
    torch.manual_seed(0)
    wrap = mhc.MHCResidualWrapper(128, n, branch_dropout=0.25, checkpoint_8bit=mode == "kept").to(cuda)
    res, w = torch.randn(30, 128, device=cuda), torch.ones(128, device=cuda)
    rng = wrap.branch_dropout.take((30, 128))
    fresh = torch.randn(30, 128, device=cuda)
    for prenorm, call in enumerate((lambda r, b: wrap(r, b, dropout_rng=rng),
                                    lambda r, b: wrap.forward_prenorm(r, b, w, dropout_rng=rng)[1])):
        runs = []
        for how in ("plain", True, False):
            if mode == "kept" and prenorm and how is True:
                continue  # its first run has no gradients, where the norm's kernel is another (with p = 0 too)
            r, b = res.clone().requires_grad_(True), fresh.clone().requires_grad_(True)
            out = call(r, b) if how == "plain" else checkpoint(call, r, b, use_reentrant=how)
            out.square().sum().backward()
            runs.append((out, r.grad, b.grad))
        assert all(torch.equal(a, c) for run in runs[1:] for a, c in zip(run, runs[0]))
        kept = mhc.checkpoint8_recompute(call, res, fresh.clone().requires_grad_(True), kept=2)
        assert torch.equal(kept, runs[0][0])
    b = fresh.clone().requires_grad_(True)
    out = checkpoint(wrap, res, b, use_reentrant=False)
    with pytest.raises(RuntimeError, match="take them before"):
        out.sum().backward()
    wrap.eval()
    assert torch.equal(wrap(res, fresh, dropout_rng=rng), wrap(res, fresh))


@pytest.mark.gpu
def test_numbers_of_another_place_are_refused(cuda):
    layer = mhc.StreamDropout(0.4).to(cuda)
    with pytest.raises(RuntimeError, match="rng"):
        layer(torch.ones(8, device=cuda), torch.zeros(2, device=cuda))
