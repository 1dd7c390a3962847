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


# ---------------------------------------------------------------------------
# data-parallel ranks
# ---------------------------------------------------------------------------

class Model(nn.Module):
    def __init__(self, seed, **rank):
        super().__init__()
        self.linear = nn.Linear(4, 4)
        self.drop = mhc.StreamDropout(0.5, seed, **rank)
        self.wrap = mhc.MHCResidualWrapper(8, branch_dropout=0.1, dropout_seed=seed,
                                           **{"dropout_" + k: v for k, v in rank.items()})

    def forward(self, x):
        return self.linear(x)


def _rank(rank, world, port, path, q):
    os.environ["MASTER_ADDR"] = "127.0.0.1"
    os.environ["MASTER_PORT"] = str(port)
    dist.init_process_group("gloo", rank=rank, world_size=world)
    try:
        seen = {}
        own = Model(100 + rank)
        for counter in (own.drop.counter, own.wrap.branch_dropout.counter):
            counter.state[1] = 1000 * (rank + 1)  # ragged batches: the ranks' positions differ too
        seen["own seeds"] = _step(own)
        one = Model(100, rank=rank)
        seen["one seed"] = _step(one)
        if rank == 0:
            one.drop.counter.state[1] = 77
            torch.save(one.state_dict(), path)
        dist.barrier()
        again = Model(5, rank=rank)  # every rank loads rank 0's file
        again.load_state_dict(torch.load(path))
        seen["restored"] = _step(again)
        q.put((rank, seen))
    finally:
        dist.destroy_process_group()


def _step(model):
    wrapped = nn.parallel.DistributedDataParallel(model, find_unused_parameters=True)
    for _ in range(2):
        wrapped(torch.ones(2, 4)).sum().backward()
    return [c.state.tolist() for c in (model.drop.counter, model.wrap.branch_dropout.counter)]


def test_ranks_keep_their_numbers(tmp_path):
    """Wrapped for data parallelism, whose wrapper broadcasts buffers, and restored from one
    rank's file."""
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    ctx = mp.get_context("spawn")
    q = ctx.Queue()
    procs = [ctx.Process(target=_rank, args=(r, 2, port, str(tmp_path / "model.pt"), q)) for r in range(2)]
    for p in procs:
        p.start()
    results = dict(q.get(timeout=120) for _ in procs)
    for p in procs:
        p.join(timeout=60)
        assert p.exitcode == 0
    zero, one = results[0], results[1]
    assert zero["own seeds"] == [[100, 1000]] * 2 and one["own seeds"] == [[101, 2000]] * 2
    assert zero["one seed"] == [[100, 0]] * 2
    assert one["one seed"][0][0] != 100 and one["one seed"] == [[one["one seed"][0][0], 0]] * 2
    assert zero["restored"] == [[100, 77], [100, 0]]
    assert one["restored"] == [[one["one seed"][0][0], 77], [one["one seed"][0][0], 0]]


def test_state_of_a_rank_is_saved_for_any():
    far = mhc.DropoutCounter(2 ** 63 + 5, 2 ** 64 - 9, rank=3)
    assert far.state[0].item() not in (2 ** 63 + 5 - 2 ** 64, 2 ** 63 + 8 - 2 ** 64)
    saved = far.state_dict()["state"]
    assert saved.tolist() == [2 ** 63 + 5 - 2 ** 64, -9] and list(far.state_dict()) == ["state"]
    for rank in (0, 1, 3):
        other = mhc.DropoutCounter(rank=rank)
        held = other.state
        assert other.load_state_dict(far.state_dict()).missing_keys == []
        assert other.state is held and other.state.tolist() == mhc.DropoutCounter(2 ** 63 + 5, 2 ** 64 - 9, rank=rank).state.tolist()
    layer = mhc.StreamDropout(0.1, 4)
    with pytest.raises(RuntimeError, match="Missing key.*counter.state"):
        layer.load_state_dict({})
    assert layer.load_state_dict({}, strict=False).missing_keys == ["counter.state"]
    with pytest.raises(RuntimeError, match="Unexpected key.*counter.other"):
        layer.load_state_dict({**layer.state_dict(), "counter.other": saved})
    with pytest.raises(RuntimeError, match="size mismatch for counter.state"):
        layer.load_state_dict({"counter.state": torch.zeros(3, dtype=torch.int64)})
    layer.load_state_dict({"counter.state": torch.tensor([8, 9])}, assign=True)
    assert layer.counter.state.tolist() == [8, 9]
    assert layer.to("meta").counter.state.is_meta and list(layer.buffers()) == []
    assert len({tuple(mhc.DropoutCounter(s, rank=r).state.tolist()) for s in range(50) for r in range(50)}) == 2500


def test_counter_pickled_as_a_buffer():
    """Modules pickled when the state was one."""
    old = mhc.DropoutCounter(6, 7)
    state = old.__dict__.copy()
    del state["rank"]
    state["_buffers"] = {"state": state.pop("state")}
    new = mhc.DropoutCounter.__new__(mhc.DropoutCounter)
    new.__setstate__(state)
    assert new.state.tolist() == [6, 7] and new.rank == 0 and list(new.buffers()) == []
    assert new.state_dict()["state"].tolist() == [6, 7]
    assert copy.deepcopy(new).state.tolist() == [6, 7]


@pytest.mark.gpu
def test_ranks_drop_other_places(cuda):
    layers = [mhc.StreamDropout(0.5, 3, rank=r).to(cuda) for r in range(4)]
    x = torch.ones(4096, device=cuda)
    assert layers[0].counter.state.is_cuda
    masks = [layer(x) != 0 for layer in layers]
    for i in range(4):
        for j in range(i):  # 4096 coins each: half of them meet, give or take 6 deviations
            assert abs((masks[i] == masks[j]).float().mean().item() - 0.5) < 6 * 0.5 / 64
    saved = [layer.state_dict()["counter.state"].tolist() for layer in layers]
    assert saved == [[3, 512]] * 4  # one file for all
    held = layers[2].counter.state.data_ptr()
    layers[2].load_state_dict({"counter.state": torch.tensor([3, 0])})
    assert layers[2].counter.state.data_ptr() == held and torch.equal(layers[2](x) != 0, masks[2])
