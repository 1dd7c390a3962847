"""Residual addition and RMSNorm in one pass, with dropout of the branch and an
output in 8 bits.

The blocks of a model that keep a plain residual stream beside the mHC ones run
``hidden = residual + dropout(branch)`` and normalise the sum for the next
branch.  ``add_rmsnorm`` does both in one pass, forward and backward, and can
write the output's 8-bit checkpoint with it, which ``linear_checkpoint8`` then
need not pack.  ``add_rmsnorm_quantized`` is the serving form: the output as
8-bit codes with scales, without padding; ``Coded8.unpack`` restores it.  The reference has
no counterpart (it normalises by itself, ops.py:87-136).
"""

from __future__ import annotations

from typing import Optional

import torch
from torch.autograd.function import once_differentiable

from . import _C
from .checkpoint8 import _FLOATS, _check_float, _dense, _empty, _weight
from .counter_dropout import Rng, _drop, _source, dropout_fwd
from .ops import _launch, _require_cuda

GROUP = 128
_CODES = (torch.float8_e4m3fn, torch.int8)


def _check_inputs(what, residual, branch, weight):
    try:  # all at once, for the calls that are right: a small call's time is the host's
        if (residual.is_cuda and residual.device == branch.device == weight.device and residual.dtype in _FLOATS
                and branch.dtype in _FLOATS and residual.shape == branch.shape and weight.dim() == 1
                and residual.size(-1) == weight.size(0) > 0):
            return
    except (AttributeError, IndexError):
        pass
    _require_cuda(what, residual, branch, weight)
    _check_float(what, "residual", residual)
    _check_float(what, "branch", branch)
    if residual.dim() == 0 or residual.size(-1) == 0:
        raise RuntimeError(f"{what}: residual must have a last dimension of at least 1")
    if branch.shape != residual.shape:
        raise RuntimeError(f"{what}: residual and branch must have one shape (got {tuple(residual.shape)} and "
                           f"{tuple(branch.shape)})")
    if weight.dim() != 1 or weight.size(0) != residual.size(-1):
        raise RuntimeError(f"{what}: weight must be 1D with size equal to hidden_dim")


def _dropout_args(what, p, rng, device):
    drop = _drop(what, p)
    if drop == 0:
        return 0, None, 0, 0
    if rng is None:
        raise RuntimeError(f"{what}: dropout needs rng = (seed, position)")
    return (drop, *_source(what, rng, device))


def _workspace_bytes(rows, cols):
    return _C.load().mhc_add_rmsnorm_bwd_workspace_bytes(rows, cols)


def add_rmsnorm_fwd(residual: torch.Tensor, branch: torch.Tensor, weight: torch.Tensor, eps: float = 1e-5,
                    p: float = 0.0, rng: Optional[Rng] = None, keep: bool = False):
    """(hidden, out, rms, kept): hidden = residual + dropout(branch, p, rng) in
    residual's type, out its RMSNorm times weight in branch's type, rms [rows] fp32,
    kept = ``checkpoint8_pack(out)`` if ``keep``, else None.  residual and branch
    [..., C] are float32 or bfloat16 each; the norm is of hidden as returned."""
    what = "add_rmsnorm_fwd"
    _check_inputs(what, residual, branch, weight)
    drop = _dropout_args(what, p, rng, residual.device)
    r, b, w = _dense(residual), _dense(branch), _weight(weight)
    hidden = torch.empty_like(r)
    out = torch.empty_like(b)
    kept = _empty(out.shape, out.dtype, out.device) if keep else None
    cols = r.size(-1)
    rows = r.numel() // cols
    rms = torch.empty(rows, dtype=torch.float32, device=r.device)
    _launch("mhc_add_rmsnorm_fwd", r.device, r.data_ptr(), r.dtype == torch.bfloat16, b.data_ptr(),
            b.dtype == torch.bfloat16, w.data_ptr(), hidden.data_ptr(), out.data_ptr(), rms.data_ptr(),
            kept.codes.data_ptr() if keep else None, kept.exponents.data_ptr() if keep else None, rows, cols, float(eps),
            *drop)
    return hidden, out, rms, kept


def add_rmsnorm_bwd(grad_hidden: Optional[torch.Tensor], grad_out: torch.Tensor, hidden: torch.Tensor,
                    weight: torch.Tensor, rms: torch.Tensor, p: float = 0.0, rng: Optional[Rng] = None):
    """(grad of residual in hidden's type, grad of branch in grad_out's, grad of
    weight fp32) from the gradients of hidden (None: zero) and out.  Without dropout
    and with one type the first two are one tensor."""
    what = "add_rmsnorm_bwd"
    _check_inputs(what, hidden, grad_out, weight)
    dev = hidden.device
    cols = hidden.size(-1)
    rows = hidden.numel() // cols
    if rms.device != dev or rms.numel() != rows:
        raise RuntimeError(f"{what}: rms must be [{rows}] on {dev}")
    drop = _dropout_args(what, p, rng, dev)
    gh = None
    if grad_hidden is not None:
        if grad_hidden.device != dev:
            raise RuntimeError(f"{what}: grad_hidden must be on {dev}")
        if grad_hidden.shape != hidden.shape or grad_hidden.dtype != hidden.dtype:
            raise RuntimeError(f"{what}: grad_hidden must have hidden's shape and type")
        gh = _dense(grad_hidden)
    h, g, w, r = _dense(hidden), _dense(grad_out), _weight(weight), _weight(rms)
    gr = torch.empty_like(h)
    one = drop[0] == 0 and g.dtype == h.dtype
    gb = gr if one else torch.empty_like(g)
    gw = torch.empty(cols, dtype=torch.float32, device=dev)
    ws = torch.empty(_workspace_bytes(rows, cols), dtype=torch.uint8, device=dev)
    _launch("mhc_add_rmsnorm_bwd", dev, 0 if gh is None else gh.data_ptr(), g.data_ptr(), h.data_ptr(),
            h.dtype == torch.bfloat16, g.dtype == torch.bfloat16, w.data_ptr(), r.data_ptr(), gr.data_ptr(),
            0 if one else gb.data_ptr(), gw.data_ptr(), rows, cols, *drop, ws.data_ptr(), ws.numel())
    return gr, gb, gw


class AddRMSNormFunction(torch.autograd.Function):
    """Residual addition and RMSNorm that saves the hidden state it returns, and no
    mask."""

    @staticmethod
    def forward(ctx, residual, branch, weight, eps, p, rng, keep):
        hidden, out, rms, kept = add_rmsnorm_fwd(residual, branch, weight, eps, p, rng, keep)
        ctx.p, ctx.rng = p, None
        saved = [hidden, weight, rms]
        if _drop("add_rmsnorm", p):
            if torch.is_tensor(rng):
                saved.append(rng)
            else:
                ctx.rng = tuple(rng)
        ctx.save_for_backward(*saved)
        ctx.set_materialize_grads(False)
        ctx.out_dtype = out.dtype
        return (hidden, out, kept) if keep else (hidden, out)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_hidden, grad_out, *_):
        hidden, weight, rms, *rng = ctx.saved_tensors
        if grad_hidden is None and grad_out is None:
            return (None,) * 7
        rng = rng[0] if rng else ctx.rng
        if grad_out is None:  # the norm, which may have no gradient (rows of zeros, infinities), has no part in it
            gb = grad_hidden
            if rng is not None:  # the product in fp32, rounded once
                gb = dropout_fwd(gb if gb.dtype == ctx.out_dtype else gb.float(), ctx.p, rng)
            return grad_hidden, gb.to(ctx.out_dtype), torch.zeros_like(weight), None, None, None, None
        gr, gb, gw = add_rmsnorm_bwd(grad_hidden, grad_out, hidden, weight, rms, ctx.p, rng)
        return gr, gb, gw.to(weight.dtype), None, None, None, None


def add_rmsnorm(residual: torch.Tensor, branch: torch.Tensor, weight: torch.Tensor, eps: float = 1e-5,
                p: float = 0.0, rng: Optional[Rng] = None, keep: bool = False):
    """(hidden, out): hidden = residual + dropout(branch, p, rng) in residual's type,
    out = hidden / sqrt(mean hidden**2 + eps) * weight in branch's type, with
    autograd.  ``rng`` as for ``dropout``; it is needed where p > 0.  With ``keep``
    (hidden, out, kept): out in 8 bits too, for ``linear_checkpoint8(out, ...,
    kept=kept)``."""
    return AddRMSNormFunction.apply(residual, branch, weight, eps, p, rng, keep)


class Coded8:
    """A tensor in 8-bit codes with scales.

    Args:
        codes: float8_e4m3fn or int8, contiguous [..., C]
        scales: float32; one a row [rows, 1], or one for each 128 columns
            [rows, ceil(C / 128)] (the last group may be shorter)
    A code stands for code * scale."""

    __slots__ = ("codes", "scales")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor):
        _require_cuda("Coded8", codes, scales)
        if codes.dtype not in _CODES or codes.dim() == 0 or codes.size(-1) == 0 or not codes.is_contiguous():
            raise RuntimeError("Coded8: codes must be a contiguous float8_e4m3fn or int8 tensor of at least one column")
        rows = codes.numel() // codes.size(-1)
        groups = -(-codes.size(-1) // GROUP)
        if scales.dtype != torch.float32 or not scales.is_contiguous() or scales.shape not in ((rows, 1), (rows, groups)):
            raise RuntimeError(f"Coded8: scales must be contiguous float32 [{rows}, 1] or [{rows}, {groups}]")
        self.codes, self.scales = codes, scales

    def unpack(self, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
        """code * scale in ``dtype`` (float32 or bfloat16)."""
        what = "Coded8.unpack"
        if dtype not in (torch.float32, torch.bfloat16):
            raise RuntimeError(f"{what}: dtype must be float32 or bfloat16 (got {dtype})")
        codes = self.codes
        out = torch.empty_like(codes, dtype=dtype)
        cols = codes.size(-1)
        _launch("mhc_coded8_unpack", codes.device, codes.data_ptr(), codes.dtype == torch.int8, self.scales.data_ptr(),
                self.scales.size(1) > 1, out.data_ptr(), dtype == torch.bfloat16, codes.numel() // cols, cols)
        return out

    def __repr__(self):
        return f"Coded8(shape={tuple(self.codes.shape)}, codes={self.codes.dtype}, scales={tuple(self.scales.shape)})"


def add_rmsnorm_quantized(residual: torch.Tensor, branch: torch.Tensor, weight: torch.Tensor, eps: float = 1e-5,
                          codes: torch.dtype = torch.float8_e4m3fn, group: Optional[int] = None):
    """(hidden, Coded8 of the output), one pass, without gradients: hidden =
    residual + branch, the output is ``add_rmsnorm``'s before it is rounded.
    ``codes``: torch.float8_e4m3fn or torch.int8; ``group``: None for a scale a row,
    128 for one for each 128 columns.  scale = max(largest |out| / 448 (127 for
    int8), 2**-100); a row or group with an infinity or a NaN, also of hidden * weight
    in fp32, stands for NaNs."""
    what = "add_rmsnorm_quantized"
    _check_inputs(what, residual, branch, weight)
    if codes not in _CODES:
        raise RuntimeError(f"{what}: codes must be torch.float8_e4m3fn or torch.int8 (got {codes})")
    if group not in (None, GROUP):
        raise RuntimeError(f"{what}: group must be None or {GROUP} (got {group})")
    if torch.is_grad_enabled() and (residual.requires_grad or branch.requires_grad or weight.requires_grad):
        raise RuntimeError(f"{what}: it has no gradient: call it under torch.no_grad(), or use add_rmsnorm")
    r, b, w = _dense(residual), _dense(branch), _weight(weight)
    hidden = torch.empty_like(r)
    coded = object.__new__(Coded8)
    coded.codes = torch.empty_like(r, dtype=codes)
    cols = r.size(-1)
    rows = r.numel() // cols
    coded.scales = torch.empty(rows, 1 if group is None else -(-cols // GROUP), dtype=torch.float32, device=r.device)
    _launch("mhc_add_rmsnorm_coded", r.device, r.data_ptr(), r.dtype == torch.bfloat16, b.data_ptr(),
            b.dtype == torch.bfloat16, w.data_ptr(), hidden.data_ptr(), coded.codes.data_ptr(), codes == torch.int8,
            coded.scales.data_ptr(), group is not None, rows, cols, float(eps))
    return hidden, coded
