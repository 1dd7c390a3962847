"""Log probabilities of given tokens, with entropy and the most likely
alternatives, and the gradient of the logits.

The end of a step beside ``StreamEmbedding`` at its start: ``-logprob`` of the
next tokens is the training loss, the entropy its regulariser, and the
alternatives are what a model answers with.  One pass over the logits, in the
type they have; nothing of their size is kept or written but the gradient, as long as
they are one matrix of rows: a contiguous tensor, or two dimensions with any distance of
rows.  Others, ``logits[:, :-1]`` of three dimensions among them, are copied in each
pass.  The reference has no counterpart (its layers end at the streams).
"""

from __future__ import annotations

from typing import NamedTuple, Optional

import torch
from torch.autograd.function import once_differentiable

from .checkpoint8 import _FLOATS, _check_float, _dense, _rows2d, _weight
from .ops import _launch, _ptr, _require_cuda

MOST_TOP = 32
_INTS = (torch.int64, torch.int32)


class TokenLogprobs(NamedTuple):
    """Results of ``token_logprobs``; ... are the logits' leading dimensions."""
    logprob: torch.Tensor  # [...] fp32
    entropy: torch.Tensor  # [...] fp32
    top_logprob: Optional[torch.Tensor]  # [..., top] fp32, largest first; None without alternatives
    top_id: Optional[torch.Tensor]  # [..., top] int64
    stats: Optional[torch.Tensor] = None  # [rows, 2] fp32, for token_logprobs_bwd


def _check(what, logits, targets, top):
    try:  # all at once, for the calls that are right: a small call's time is the host's
        if (logits.is_cuda and logits.device == targets.device and logits.dtype in _FLOATS and targets.dtype in _INTS
                and targets.shape == logits.shape[:-1] and logits.dim() and 0 <= top <= MOST_TOP
                and max(top, 1) <= logits.size(-1)):
            return
    except AttributeError:
        pass
    _require_cuda(what, logits, targets)
    _check_float(what, "logits", logits)
    if logits.dim() == 0 or logits.size(-1) == 0:
        raise RuntimeError(f"{what}: logits must be [..., vocab] with a vocabulary of at least 1")
    if targets.dtype not in _INTS:
        raise RuntimeError(f"{what}: targets must be int64 or int32 (got {targets.dtype})")
    if targets.shape != logits.shape[:-1]:
        raise RuntimeError(f"{what}: targets must have the logits' leading dimensions {tuple(logits.shape[:-1])} "
                           f"(got {tuple(targets.shape)})")
    if not 0 <= top <= min(MOST_TOP, logits.size(-1)):
        raise RuntimeError(f"{what}: top must be in [0, {min(MOST_TOP, logits.size(-1))}] (got {top})")


def token_logprobs_fwd(logits: torch.Tensor, targets: torch.Tensor, top: int = 0,
                       ignore_index: int = -100) -> TokenLogprobs:
    """``token_logprobs`` without autograd, with the ``stats`` that its backward takes."""
    what = "token_logprobs"
    _check(what, logits, targets, top)
    x, stride = _rows2d(logits)
    t = _dense(targets)
    rows, vocab = x.shape
    lead, dev = t.shape, x.device
    logprob = torch.empty_like(t, dtype=torch.float32)
    entropy = torch.empty_like(logprob)
    stats = torch.empty(rows, 2, dtype=torch.float32, device=dev)
    top_logprob = top_id = None
    values = ids = 0
    if top:
        top_logprob = torch.empty(*lead, top, dtype=torch.float32, device=dev)
        top_id = torch.empty(*lead, top, dtype=torch.int64, device=dev)
        values, ids = top_logprob.data_ptr(), top_id.data_ptr()
    _launch("mhc_token_logprobs_fwd", dev, x.data_ptr(), x.dtype == torch.bfloat16, stride, t.data_ptr(),
            t.dtype == torch.int64, ignore_index, logprob.data_ptr(), entropy.data_ptr(), values, ids, stats.data_ptr(),
            rows, vocab, top)
    return TokenLogprobs(logprob, entropy, top_logprob, top_id, stats)


def token_logprobs_bwd(logits: torch.Tensor, targets: torch.Tensor, result: TokenLogprobs,
                       grad_logprob: Optional[torch.Tensor] = None, grad_entropy: Optional[torch.Tensor] = None,
                       grad_top: Optional[torch.Tensor] = None, ignore_index: int = -100) -> torch.Tensor:
    """Gradient of the logits, contiguous and in their type, from the gradients of
    the log probabilities, of the entropies and of the alternatives' log
    probabilities (None: zero); ``result`` is ``token_logprobs_fwd``'s."""
    what = "token_logprobs_bwd"
    top = 0
    if grad_top is not None:
        if result.top_id is None or grad_top.shape != result.top_id.shape:
            raise RuntimeError(f"{what}: grad_top must have top_id's shape")
        top = grad_top.size(-1)
    _check(what, logits, targets, top)
    x, stride = _rows2d(logits)
    rows, vocab = x.shape
    if result.stats is None or result.stats.shape != (rows, 2) or result.entropy.numel() != rows or \
            (top and (result.top_id.shape != (*targets.shape, top) or result.top_id.dtype != torch.int64)):
        raise RuntimeError(f"{what}: result must be token_logprobs_fwd's for these logits")
    dev = x.device
    for t in (result.stats, result.entropy, result.top_id if top else None, grad_logprob, grad_entropy, grad_top):
        if t is not None and t.device != dev:
            _require_cuda(what, x, t)
    grads = []
    for name, g in (("grad_logprob", grad_logprob), ("grad_entropy", grad_entropy), ("grad_top", grad_top)):
        if g is not None:
            if name != "grad_top" and g.shape != targets.shape:
                raise RuntimeError(f"{what}: {name} must have targets' shape")
            g = _weight(g)
        grads.append(g)
    t = _dense(targets)
    ids = _dense(result.top_id) if top else None
    stats, entropy = _weight(result.stats), _weight(result.entropy)
    gx = torch.empty_like(logits, memory_format=torch.contiguous_format)
    _launch("mhc_token_logprobs_bwd", x.device, x.data_ptr(), x.dtype == torch.bfloat16, stride, t.data_ptr(),
            t.dtype == torch.int64, int(ignore_index), stats.data_ptr(), entropy.data_ptr(), _ptr(ids), _ptr(grads[0]),
            _ptr(grads[1]), _ptr(grads[2]), gx.data_ptr(), rows, vocab, top)
    return gx


class TokenLogprobsFunction(torch.autograd.Function):
    """Log probabilities that save the logits and two numbers a row."""

    @staticmethod
    def forward(ctx, logits, targets, top, ignore_index):
        r = token_logprobs_fwd(logits, targets, top, ignore_index)
        saved = [logits, targets, r.entropy, r.stats]
        if top:
            saved.append(r.top_id)
            ctx.mark_non_differentiable(r.top_id)
        ctx.save_for_backward(*saved)
        ctx.ignore_index = ignore_index
        ctx.set_materialize_grads(False)
        return r.logprob, r.entropy, r.top_logprob, r.top_id

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_logprob, grad_entropy, grad_top, _):
        logits, targets, entropy, stats, *ids = ctx.saved_tensors
        if grad_logprob is None and grad_entropy is None and grad_top is None:
            return None, None, None, None
        result = TokenLogprobs(None, entropy, None, ids[0] if ids else None, stats)
        gx = token_logprobs_bwd(logits, targets, result, grad_logprob, grad_entropy, grad_top, ctx.ignore_index)
        return gx, None, None, None


def token_logprobs(logits: torch.Tensor, targets: torch.Tensor, top: int = 0, ignore_index: int = -100) -> TokenLogprobs:
    """Log probability of ``targets`` [...] (int64 or int32) under ``logits``
    [..., vocab] (float32 or bfloat16), the distributions' entropies, and the ``top``
    (at most 32) most likely tokens with their log probabilities, ties to the lowest
    id; with autograd for all but the ids.

    A target equal to ``ignore_index`` has log probability 0 and gives no gradient;
    any other outside the vocabulary has NaN, and so has the gradient through it
    (entropy and alternatives do not depend on it).  A logit of -inf is a token that
    cannot come; a row of nothing else has log probabilities -inf, entropy 0 and no
    gradient."""
    return TokenLogprobs(*TokenLogprobsFunction.apply(logits, targets, top, ignore_index))
