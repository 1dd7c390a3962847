"""Activation checkpoints in 8 bits and their use in the backward pass.

With n residual streams a step keeps n times a plain model's activations.  A
``Checkpoint8`` keeps a tensor in 33/32 bytes a value (fp32: 3.9 times less):
int8 codes and a power-of-two step for each block of 32 values along the last
dimension.  The backward operators take the codes as they are:

* ``rmsnorm_checkpoint8`` -- RMSNorm that packs its input in its forward pass;
* ``linear_checkpoint8`` -- linear layer whose weight gradient is formed from
  the packed input on the tensor cores;
* ``checkpoint8_recompute`` -- any function of tensors: keeps its input packed
  and runs it again; ``MHCLayer(checkpoint_8bit=True)`` keeps its streams so.

Each gradient is the exact gradient formula evaluated at the restored input;
it is not differentiable again (autograd raises).
The reference has no counterpart (it saves bf16 copies, ops.py:394-470).
"""

from __future__ import annotations

import math
from typing import Optional, Sequence

import torch
from torch.autograd.function import once_differentiable

from .counter_dropout import no_new_numbers
from .ops import _f32, _launch, _lib, _require_cuda, _workspace

BLOCK, PITCH = 32, 128
_FLOATS = (torch.float32, torch.bfloat16)


def _pitch(cols):
    return -(-cols // PITCH) * PITCH


class Checkpoint8:
    """A tensor kept in 8 bits.

    Args:
        codes: int8 [rows, pitch], pitch = 128 * ceil(cols / 128); rows are the
            leading dimensions of ``shape`` flattened, cols its last
        exponents: uint8 [rows, pitch / 32]; code c of block b stands for
            c * 2**(exponents[b] - 127), and a block with exponent 255 for NaNs
        shape: shape of the kept tensor
        dtype: type it had (what ``unpack`` returns by default)
    """

    __slots__ = ("codes", "exponents", "shape", "dtype", "rows", "cols")

    def __init__(self, codes: torch.Tensor, exponents: torch.Tensor, shape: Sequence[int], dtype: torch.dtype):
        self.shape = torch.Size(shape)
        if len(self.shape) == 0 or self.shape[-1] == 0:
            raise RuntimeError("Checkpoint8: shape must have a last dimension of at least 1")
        if dtype not in _FLOATS:
            raise RuntimeError(f"Checkpoint8: dtype must be float32 or bfloat16 (got {dtype})")
        _require_cuda("Checkpoint8", codes, exponents)
        self.cols = self.shape[-1]
        self.rows = rows = math.prod(self.shape[:-1])
        pitch = _pitch(self.cols)
        if codes.dtype != torch.int8 or codes.shape != (rows, pitch) or not codes.is_contiguous():
            raise RuntimeError(f"Checkpoint8: codes must be a contiguous int8 [{rows}, {pitch}] tensor")
        if exponents.dtype != torch.uint8 or exponents.shape != (rows, pitch // BLOCK) \
                or not exponents.is_contiguous():
            raise RuntimeError(f"Checkpoint8: exponents must be a contiguous uint8 [{rows}, {pitch // BLOCK}] tensor")
        self.codes, self.exponents, self.dtype = codes, exponents, dtype

    def unpack(self, dtype: Optional[torch.dtype] = None) -> torch.Tensor:
        return checkpoint8_unpack(self, dtype)

    def __repr__(self):
        return f"Checkpoint8(shape={tuple(self.shape)}, dtype={self.dtype})"


def _empty(shape, dtype, device):
    c = object.__new__(Checkpoint8)
    c.shape, c.dtype, c.cols = shape, dtype, shape[-1]
    c.rows = rows = math.prod(shape[:-1])
    pitch = _pitch(c.cols)
    c.codes = torch.empty(rows, pitch, dtype=torch.int8, device=device)
    c.exponents = torch.empty(rows, pitch // BLOCK, dtype=torch.uint8, device=device)
    return c


def _rows2d(t):
    """t as [rows, cols] with unit column stride and rows apart by at least
    cols: a view where it can be one.  (tensor, row stride)"""
    cols = t.size(-1)
    if t.dim() == 2 and (t.stride(1) == 1 or cols == 1) and t.stride(0) >= cols:
        return t, t.stride(0)
    return t.detach().reshape(-1, cols).contiguous(), cols


def _dense(t):
    return t if t.is_contiguous() else t.detach().contiguous()


def _weight(t):
    return t if t.dtype == torch.float32 and t.is_contiguous() else _f32(t)


def _check_float(what, name, t):
    if t.dtype not in _FLOATS:
        raise RuntimeError(f"{what}: {name} must be float32 or bfloat16 (got {t.dtype})")


def checkpoint8_pack(x: torch.Tensor) -> Checkpoint8:
    """Keep x (float32 or bfloat16, blocks along the last dimension) in 8 bits."""
    what = "checkpoint8_pack"
    _require_cuda(what, x)
    _check_float(what, "x", x)
    if x.dim() == 0 or x.size(-1) == 0:
        raise RuntimeError(f"{what}: x must have a last dimension of at least 1")
    x2, stride = _rows2d(x)
    kept = _empty(x.shape, x.dtype, x.device)
    _launch("mhc_checkpoint8_pack", x.device, x2.data_ptr(), x.dtype == torch.bfloat16, stride,
            kept.codes.data_ptr(), kept.exponents.data_ptr(), x2.size(0), x2.size(1))
    return kept


def checkpoint8_unpack(kept: Checkpoint8, dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """The kept tensor's restored values (exact in both types)."""
    what = "checkpoint8_unpack"
    dtype = kept.dtype if dtype is None else dtype
    if dtype not in _FLOATS:
        raise RuntimeError(f"{what}: dtype must be float32 or bfloat16 (got {dtype})")
    dev = kept.codes.device
    out = torch.empty(kept.shape, dtype=dtype, device=dev)
    _launch("mhc_checkpoint8_unpack", dev, kept.codes.data_ptr(), kept.exponents.data_ptr(), out.data_ptr(),
            dtype == torch.bfloat16, kept.rows, kept.cols)
    return out


# =============================================================================
# RMSNorm
# =============================================================================

def rmsnorm_checkpoint8_fwd(inp: torch.Tensor, weight: torch.Tensor, eps: float = 1e-5):
    """(out in inp's type, rms [rows] fp32, inp kept in 8 bits), one pass over inp [..., C]."""
    what = "rmsnorm_checkpoint8_fwd"
    _require_cuda(what, inp, weight)
    _check_float(what, "inp", inp)
    if inp.dim() == 0 or inp.size(-1) == 0:
        raise RuntimeError(f"{what}: inp must have a last dimension of at least 1")
    if weight.dim() != 1 or weight.size(0) != inp.size(-1):
        raise RuntimeError("Weight must be 1D with size equal to hidden_dim")
    x, w = _dense(inp), _weight(weight)
    kept = _empty(x.shape, x.dtype, x.device)
    out = torch.empty_like(x, requires_grad=False)
    rows = kept.rows
    rms = torch.empty(rows, dtype=torch.float32, device=x.device)
    _launch("mhc_rmsnorm_checkpoint8_fwd", x.device, x.data_ptr(), x.dtype == torch.bfloat16, w.data_ptr(),
            out.data_ptr(), rms.data_ptr(), kept.codes.data_ptr(), kept.exponents.data_ptr(), rows, kept.cols,
            float(eps))
    return out, rms, kept


def rmsnorm_checkpoint8_bwd(grad_out: torch.Tensor, kept: Checkpoint8, weight: torch.Tensor, rms: torch.Tensor):
    """(grad of the input in grad_out's type, grad of the weight fp32) at the restored input."""
    what = "rmsnorm_checkpoint8_bwd"
    _require_cuda(what, grad_out, kept.codes, weight, rms)
    _check_float(what, "grad_out", grad_out)
    if grad_out.shape != kept.shape:
        raise RuntimeError(f"{what}: grad_out must have the kept input's shape {tuple(kept.shape)}")
    rows, cols = kept.rows, kept.cols
    if weight.shape != (cols,) or rms.numel() != rows:
        raise RuntimeError(f"{what}: weight must be [{cols}] and rms [{rows}]")
    g, w, r = _dense(grad_out), _weight(weight), _weight(rms)
    gx = torch.empty_like(g)
    gw = torch.empty(cols, dtype=torch.float32, device=g.device)
    ws = _workspace(_lib.mhc_rmsnorm_checkpoint8_bwd_workspace_bytes(rows, cols), g.device)
    _launch("mhc_rmsnorm_checkpoint8_bwd", g.device, g.data_ptr(), g.dtype == torch.bfloat16, kept.codes.data_ptr(),
            kept.exponents.data_ptr(), w.data_ptr(), r.data_ptr(), gx.data_ptr(), gw.data_ptr(), rows, cols,
            ws.data_ptr(), ws.numel())
    return gx, gw


class RMSNormCheckpoint8Function(torch.autograd.Function):
    """RMSNorm that saves its input in 8 bits."""

    @staticmethod
    def forward(ctx, inp, weight, eps=1e-5):
        out, rms, kept = rmsnorm_checkpoint8_fwd(inp, weight, eps)
        ctx.save_for_backward(kept.codes, kept.exponents, weight, rms)
        ctx.kept = (kept.shape, kept.dtype)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_out):
        codes, exponents, weight, rms = ctx.saved_tensors
        kept = Checkpoint8(codes, exponents, *ctx.kept)
        gx, gw = rmsnorm_checkpoint8_bwd(grad_out, kept, weight, rms)
        return gx.to(kept.dtype), gw.to(weight.dtype), None


def rmsnorm_checkpoint8(inp: torch.Tensor, weight: torch.Tensor, eps: float = 1e-5) -> torch.Tensor:
    """RMS normalization over the last dimension (float32 or bfloat16, result in
    the same type) whose backward reads the input from 8 bits."""
    return RMSNormCheckpoint8Function.apply(inp, weight, eps)


# =============================================================================
# Linear layer
# =============================================================================

def checkpoint8_weight_grad(grad_out: torch.Tensor, kept: Checkpoint8,
                            dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """grad_out^T xh [out_features, in_features] in ``dtype``: grad_out
    [..., out_features] float32 or bfloat16, xh the kept input [..., in_features].
    fp32 sums; a float32 grad_out is used in full precision."""
    what = "checkpoint8_weight_grad"
    _require_cuda(what, grad_out, kept.codes)
    _check_float(what, "grad_out", grad_out)
    if dtype not in _FLOATS:
        raise RuntimeError(f"{what}: dtype must be float32 or bfloat16 (got {dtype})")
    if grad_out.dim() < 1 or grad_out.shape[:-1] != kept.shape[:-1] or grad_out.size(-1) == 0:
        raise RuntimeError(f"{what}: grad_out must be {tuple(kept.shape[:-1])} + [out_features] "
                           f"(got {tuple(grad_out.shape)})")
    g, stride = _rows2d(grad_out)
    T, O, K = kept.rows, g.size(1), kept.cols
    gw = torch.empty(O, K, dtype=dtype, device=g.device)
    g16, w16 = g.dtype == torch.bfloat16, dtype == torch.bfloat16
    aligned = g16 and stride % 8 == 0 and g.data_ptr() % 16 == 0
    ws = _workspace(_lib.mhc_checkpoint8_weight_grad_workspace_bytes(T, O, K, g16, aligned), g.device)
    _launch("mhc_checkpoint8_weight_grad", g.device, g.data_ptr(), g16, stride, kept.codes.data_ptr(),
            kept.exponents.data_ptr(), gw.data_ptr(), w16, T, O, K, ws.data_ptr(), ws.numel())
    return gw


class LinearCheckpoint8Function(torch.autograd.Function):
    """x W^T (+ b) that saves x in 8 bits.  The two plain products (forward, and
    the gradient of x, which needs no x) are torch's."""

    @staticmethod
    def forward(ctx, x, weight, bias, kept=None):
        if kept is None:
            kept = checkpoint8_pack(x)
        ctx.save_for_backward(kept.codes, kept.exponents, weight)
        ctx.kept = (kept.shape, kept.dtype)
        ctx.bias_dtype = None if bias is None else bias.dtype
        return torch.nn.functional.linear(x, weight, bias)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_out):
        codes, exponents, weight = ctx.saved_tensors
        gx = gw = gb = None
        if ctx.needs_input_grad[0]:
            gx = grad_out @ weight
        if ctx.needs_input_grad[1]:
            gw = checkpoint8_weight_grad(grad_out, Checkpoint8(codes, exponents, *ctx.kept), weight.dtype)
        if ctx.needs_input_grad[2]:
            gb = grad_out.reshape(-1, grad_out.size(-1)).sum(0, dtype=torch.float32).to(ctx.bias_dtype)
        return gx, gw, gb, None


def linear_checkpoint8(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None,
                       kept: Optional[Checkpoint8] = None) -> torch.Tensor:
    """``torch.nn.functional.linear`` (x, weight and bias of one type, float32 or
    bfloat16) that keeps x in 8 bits for the weight's gradient, and nothing of x
    where the weight needs none.  ``kept`` is x in 8 bits where the caller has it
    (``add_rmsnorm(..., keep=True)``): x is then not packed again.  Under autocast
    the three are cast to its type first, as for the plain layer."""
    _require_cuda("linear_checkpoint8", x, weight)
    if kept is not None and (kept.shape != x.shape or kept.codes.device != x.device):
        raise RuntimeError(f"linear_checkpoint8: kept must be x in 8 bits: {tuple(x.shape)} on {x.device}")
    if torch.is_autocast_enabled("cuda"):
        dtype = torch.get_autocast_dtype("cuda")
        with torch.autocast("cuda", enabled=False):
            return linear_checkpoint8(x.to(dtype), weight.to(dtype), None if bias is None else bias.to(dtype), kept)
    _check_float("linear_checkpoint8", "x", x)
    if weight.dim() != 2:
        raise RuntimeError(f"linear_checkpoint8: weight must be [out_features, in_features] (got {tuple(weight.shape)})")
    if weight.dtype != x.dtype or (bias is not None and bias.dtype != x.dtype):
        raise RuntimeError("linear_checkpoint8: x, weight and bias must have one type")
    if not (torch.is_grad_enabled() and weight.requires_grad):  # nobody will read the codes
        return torch.nn.functional.linear(x, weight, bias)
    return LinearCheckpoint8Function.apply(x, weight, bias, kept)


# =============================================================================
# Recomputation from 8 bits
# =============================================================================

def _forget(tensor):
    """Keep nothing of a tensor that a graph wants to save."""


def _forgotten(_):
    raise RuntimeError("checkpoint8_recompute: function must not differentiate inside its forward pass")


def _holds_tensors(o):
    """Whether o is a container with tensors inside."""
    if isinstance(o, dict):
        o = o.values()
    elif not isinstance(o, (list, tuple)):
        return False
    return any(torch.is_tensor(v) or _holds_tensors(v) for v in o)


class Checkpoint8Function(torch.autograd.Function):
    """function(*tensors) that saves its first `kept` tensors in 8 bits and
    nothing of its inside; the backward restores them and runs it again."""

    @staticmethod
    def forward(ctx, function, kept, *tensors):
        packed = [checkpoint8_pack(t) for t in tensors[:kept]]
        ctx.save_for_backward(*[p for c in packed for p in (c.codes, c.exponents)], *tensors[kept:])
        ctx.function, ctx.kept = function, [(c.shape, c.dtype) for c in packed]
        ctx.autocast = dict(enabled=torch.is_autocast_enabled("cuda"), dtype=torch.get_autocast_dtype("cuda"))
        # With gradients on, as the caller has them and as the recomputation runs: a
        # function that asks for the mode (as MHCLayer does) takes one path in both,
        # and the backward differentiates what the forward returned.  The graph is
        # made for that alone: it saves nothing and goes with this call.
        inside = [t.detach().requires_grad_(n) for t, n in zip(tensors, ctx.needs_input_grad[2:])]
        with torch.enable_grad(), torch.autograd.graph.saved_tensors_hooks(_forget, _forgotten), no_new_numbers():
            out = function(*inside)
        outs = out if isinstance(out, tuple) else (out,)
        if any(map(_holds_tensors, outs)):  # autograd would hand them out without a graph
            raise RuntimeError("checkpoint8_recompute: function must return a tensor or a tuple of tensors")
        outs = tuple(o.detach() if torch.is_tensor(o) else o for o in outs)
        return outs if isinstance(out, tuple) else outs[0]

    @staticmethod
    @once_differentiable
    def backward(ctx, *grad_out):
        saved, k = ctx.saved_tensors, len(ctx.kept)
        need = ctx.needs_input_grad[2:]
        tensors = [Checkpoint8(saved[2 * i], saved[2 * i + 1], *ctx.kept[i]).unpack() for i in range(k)]
        tensors += [t.detach() for t in saved[2 * k:]]
        for t, n in zip(tensors, need):
            t.requires_grad_(n)
        with torch.enable_grad(), torch.autocast("cuda", **ctx.autocast), no_new_numbers():
            out = ctx.function(*tensors)
        outs = out if isinstance(out, tuple) else (out,)
        pairs = [(o, g) for o, g in zip(outs, grad_out) if g is not None and o.requires_grad]
        grads = iter(torch.autograd.grad([o for o, _ in pairs], [t for t, n in zip(tensors, need) if n],
                                         [g for _, g in pairs], allow_unused=True))
        return (None, None, *[next(grads) if n else None for n in need])


def checkpoint8_recompute(function, *tensors: torch.Tensor, kept: int = 1):
    """Run ``function(*tensors)`` (it returns a tensor or a tuple of them) for
    training and keep only its first ``kept`` tensors, in 8 bits (float32 or
    bfloat16); the backward restores them and recomputes.  The gradients are
    those of ``function`` at the restored tensors.  ``function`` is called again
    with the same arguments and gradients on, as in the first pass: it draws no
    random numbers but those of ``dropout`` at a given (seed, position), and what it
    differentiates by has to be among ``tensors``."""
    if not 1 <= kept <= len(tensors):
        raise RuntimeError(f"checkpoint8_recompute: kept must be in [1, {len(tensors)}] (got {kept})")
    if not (torch.is_grad_enabled() and any(t.requires_grad for t in tensors)):
        return function(*tensors)
    return Checkpoint8Function.apply(function, kept, *tensors)
