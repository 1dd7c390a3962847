"""Dropout from a counter-based generator, with a mask that is never stored.

Whether a value is dropped is a function of a seed and the value's place in a
stream of random numbers, so the backward pass draws the same mask again and
nothing is kept for it.  The same holds for ``checkpoint8_recompute``: a function
that drops by a given (seed, position) gives the same result when it runs again.
The reference has no counterpart (its layers draw no random numbers).
"""

from __future__ import annotations

import contextlib
import copy
import itertools
import math
import threading
from typing import Optional, Tuple, Union

import torch
import torch.nn as nn
from torch.autograd.function import once_differentiable

from .ops import _launch, _require_cuda

GROUP = 8  # positions are counted in groups of eight values
_running_twice = threading.local()  # .depth: functions that will run, or run, a second time
_FLOATS = (torch.float32, torch.bfloat16)
_WORD = (1 << 64) - 1
_LAYERS = 0x9E3779B97F4A7C15  # odd: between the seeds of layers that are given none, so that few meet small given ones
_RANKS = 0xD1342543DE82EF95  # odd: between the seeds of ranks
_made = itertools.count()  # such layers, in the order in which they are made

Rng = Union[Tuple[int, int], torch.Tensor]


def dropout_groups(shape) -> int:
    """Positions that a tensor of this shape takes up."""
    return -(-math.prod(shape) // GROUP)


@contextlib.contextmanager
def no_new_numbers():
    """While a function runs whose second run has to draw the same numbers."""
    _running_twice.depth = getattr(_running_twice, "depth", 0) + 1
    try:
        yield
    finally:
        _running_twice.depth -= 1


def _drop(what, p):
    p = float(p)
    if not 0.0 <= p <= 1.0:
        raise RuntimeError(f"{what}: p must be in [0, 1] (got {p})")
    return round(p * 65536)


def _source(what, rng, device):
    """(state pointer or None, seed, position) for the C entry points."""
    if torch.is_tensor(rng):
        if rng.dtype != torch.int64 or rng.shape != (2,) or not rng.is_contiguous():
            raise RuntimeError(f"{what}: rng must be (seed, position) or a contiguous int64 tensor of the two")
        if rng.device != device:
            raise RuntimeError(f"{what}: rng must be on {device} (got {rng.device})")
        return rng.data_ptr(), 0, 0
    try:
        seed, position = rng
        return None, int(seed) & _WORD, int(position) & _WORD
    except (TypeError, ValueError):
        raise RuntimeError(f"{what}: rng must be (seed, position) or a contiguous int64 tensor of the two") from None


def dropout_fwd(x: torch.Tensor, p: float, rng: Rng) -> torch.Tensor:
    """x with values dropped (zero) with probability p and the others divided by
    1 - p: float32 or bfloat16, a contiguous result.  p counts as the nearest
    multiple of 2**-16.  Applied to a gradient it is the backward pass.

    ``rng`` is (seed, position), or the two in an int64 CUDA tensor, read by the
    kernel when it runs.  Value i in row-major order is decided by number i % 8 of
    group position + i // 8 of the seed's stream; x takes up
    ``dropout_groups(x.shape)`` positions."""
    what = "dropout"
    _require_cuda(what, x)
    if x.dtype not in _FLOATS:
        raise RuntimeError(f"{what}: x must be float32 or bfloat16 (got {x.dtype})")
    drop = _drop(what, p)
    source = _source(what, rng, x.device)
    xc = x if x.is_contiguous() else x.detach().contiguous()
    out = torch.empty_like(xc)
    _launch("mhc_dropout", x.device, xc.data_ptr(), x.dtype == torch.bfloat16, out.data_ptr(), xc.numel(), drop, *source)
    return out


class DropoutFunction(torch.autograd.Function):
    """Dropout that saves where its random numbers start, and no mask."""

    @staticmethod
    def forward(ctx, x, p, rng):
        out = dropout_fwd(x, p, rng)
        ctx.p, ctx.rng = p, None
        if torch.is_tensor(rng):
            ctx.save_for_backward(rng)
        else:
            ctx.rng = tuple(rng)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_out):
        rng = ctx.rng if ctx.rng is not None else ctx.saved_tensors[0]
        return dropout_fwd(grad_out, ctx.p, rng), None, None


def dropout(x: torch.Tensor, p: float, rng: Rng) -> torch.Tensor:
    """``dropout_fwd`` with autograd.  An ``rng`` tensor must keep its value until
    the backward pass (``DropoutCounter.take`` returns one that does)."""
    return DropoutFunction.apply(x, p, rng)


def _int64(v):
    v = int(v) & _WORD
    return v - (1 << 64) if v >> 63 else v


class DropoutCounter(nn.Module):
    """Seed and position of a stream of random numbers, on the device: taking
    numbers is one small kernel and no host step, so a captured graph takes new
    ones each time it is replayed.  The state moves with the module and is saved with
    it, but is no buffer: data-parallel wrappers broadcast buffers, and every rank would
    go on with rank 0's.  Ranks that are to draw different masks take different seeds,
    or one seed and a ``rank`` each: ``rank`` shifts the seed and is not saved, so that
    every rank can load one rank's file and keeps numbers of its own.  A function that a
    checkpoint runs again has to be given its numbers, taken before it: the second run
    would take others, and ``take`` raises there."""

    rank = 0  # of modules pickled before it was an argument

    def __init__(self, seed: int = 0, position: int = 0, rank: int = 0):
        super().__init__()
        self.rank = int(rank)
        self.state = torch.tensor([_int64(int(seed) + self.rank * _RANKS), _int64(position)], dtype=torch.int64)

    def _apply(self, fn, recurse=True):
        super()._apply(fn, recurse)
        self.state = fn(self.state)
        return self

    def _save_to_state_dict(self, destination, prefix, keep_vars):
        super()._save_to_state_dict(destination, prefix, keep_vars)
        state = self.state
        if self.rank:
            state = state.clone()
            state[0] -= _int64(self.rank * _RANKS)
        destination[prefix + "state"] = state

    def _load_from_state_dict(self, state_dict, prefix, local_metadata, strict, missing_keys, unexpected_keys, error_msgs):
        name = prefix + "state"
        state = state_dict.get(name)
        super()._load_from_state_dict({k: v for k, v in state_dict.items() if k != name}, prefix, local_metadata, strict,
                                      missing_keys, unexpected_keys, error_msgs)
        if state is None:
            if strict:
                missing_keys.append(name)
        elif state.shape != self.state.shape:
            error_msgs.append(f"size mismatch for {name}: {tuple(state.shape)} in place of {tuple(self.state.shape)}")
        else:
            if local_metadata.get("assign_to_params_buffers", False):
                self.state = state.to(torch.int64, copy=True)
            else:
                self.state.copy_(state)  # in place: captured graphs hold its address
            if self.rank:
                self.state[0] += _int64(self.rank * _RANKS)

    def __setstate__(self, state):
        super().__setstate__(state)
        if "state" in self._buffers:  # of modules pickled when it was one
            self.state = self._buffers.pop("state")

    def take(self, groups: int) -> torch.Tensor:
        """(seed, position) for the next ``groups`` groups as an int64 tensor of its
        own, and the position moved past them.  Inside ``checkpoint8_recompute``, and in a
        backward pass, where ``torch.utils.checkpoint`` runs a function again, it raises:
        take them before."""
        if getattr(_running_twice, "depth", 0):
            raise RuntimeError("DropoutCounter.take: a function under checkpoint8_recompute may not take new numbers: "
                               "take them before and drop by them")
        if torch._C._current_graph_task_id() != -1:  # this thread is inside a backward pass
            raise RuntimeError("DropoutCounter.take: a function that runs again in the backward pass would draw another "
                               "mask than the first time: take them before and drop by them")
        _require_cuda("DropoutCounter.take", self.state)
        if self.state.dtype != torch.int64 or not self.state.is_contiguous():
            raise RuntimeError("DropoutCounter.take: state must be a contiguous int64 tensor")
        out = torch.empty_like(self.state)
        _launch("mhc_dropout_take", self.state.device, self.state.data_ptr(), out.data_ptr(), int(groups))
        return out


class StreamDropout(nn.Module):
    """Dropout layer over its own ``DropoutCounter``; the identity in evaluation.

    Layers of one seed drop the same places.  Without a ``seed`` each layer gets another:
    the process numbers them as they are made (the first has seed 0), and a deep copy
    of such a layer counts as one more.  The order in which a program builds its model
    decides them, not ``torch.manual_seed``, so ranks that build the same model draw the
    same masks unless each has a ``rank`` (as for the counter).  A layer restored by
    ``load_state_dict`` or unpickled goes on with the seed that was saved."""

    def __init__(self, p: float, seed: Optional[int] = None, rank: int = 0):
        super().__init__()
        _drop("StreamDropout", p)
        self.p = float(p)
        self.numbered = seed is None
        self.counter = DropoutCounter(next(_made) * _LAYERS if seed is None else seed, rank=rank)

    def __deepcopy__(self, memo):
        made = memo[id(self)] = self.__class__.__new__(self.__class__)
        made.__dict__ = copy.deepcopy(self.__dict__, memo)
        if self.__dict__.get("numbered"):  # not there in layers pickled before it was
            made.counter.state[0] = _int64(next(_made) * _LAYERS + made.counter.rank * _RANKS)
        return made

    def take(self, shape) -> Optional[torch.Tensor]:
        """Numbers for one call on a tensor of this shape, for a function that a checkpoint
        runs again; None where the layer is the identity."""
        if not self.training or self.p == 0.0:
            return None
        return self.counter.take(dropout_groups(shape))

    def forward(self, x: torch.Tensor, rng: Optional[Rng] = None) -> torch.Tensor:
        """x dropped by ``rng`` (``take``'s, or (seed, position)), by new numbers without one."""
        if not self.training or self.p == 0.0:
            return x
        if rng is None:  # replicas of torch.nn.DataParallel share the counter of the first device
            rng = self.counter.take(dropout_groups(x.shape)).to(x.device)
        return dropout(x, self.p, rng)

    def extra_repr(self) -> str:
        return f"p={self.p}"
