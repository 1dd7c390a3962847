"""Token ids -> residual streams, and the embedding table's gradient.

An mHC model carries n residual streams per token; its first layer reads
``[tokens, n, hidden]``.  ``stream_embedding`` looks the tokens' rows up and
writes all n streams in one pass, each with its own scale, and its backward
adds the streams' gradients up into the dense gradient of the table by sorted
tokens: no float atomics, bitwise reproducible.  The reference has no
counterpart (its examples start from random streams, test_layer.py).
"""

from __future__ import annotations

import ctypes
from typing import Optional, Sequence, Union

import torch
import torch.nn as nn
from torch.autograd.function import once_differentiable

from .ops import _launch, _lib, _require_cuda, _workspace

_FLOATS = (torch.float32, torch.bfloat16)
MAX_STREAMS = 32


def _scales(scale, n):
    """The n scales as they are now, for the call and for its backward pass."""
    if isinstance(scale, (int, float)):
        vals = [float(scale)] * n
    else:
        vals = [float(v) for v in scale]
        if len(vals) != n:
            raise RuntimeError(f"stream_embedding: {n} streams need {n} scales (got {len(vals)})")
    return tuple(vals)


def _check_ids(what, ids):
    if ids.dtype not in (torch.int64, torch.int32):
        raise RuntimeError(f"{what}: ids must be int64 or int32 (got {ids.dtype})")
    return ids.contiguous()


def _check_n(what, n):
    if not 1 <= int(n) <= MAX_STREAMS:
        raise RuntimeError(f"{what}: num_streams must be in [1, {MAX_STREAMS}] (got {n})")
    return int(n)


def stream_embedding_fwd(ids: torch.Tensor, weight: torch.Tensor, num_streams: int,
                         scale: Union[float, Sequence[float]] = 1.0,
                         dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """``scale_i * weight[ids]`` for each stream i: ids' shape + [n, hidden] in
    ``dtype`` (default: the table's).  An id outside the table gives NaNs."""
    what = "stream_embedding"
    _require_cuda(what, ids, weight)
    n = _check_n(what, num_streams)
    if weight.dim() != 2 or weight.dtype not in _FLOATS or not weight.is_contiguous():
        raise RuntimeError(f"{what}: weight must be a contiguous [vocab, hidden] float32 or bfloat16 tensor")
    dtype = weight.dtype if dtype is None else dtype
    if dtype not in _FLOATS:
        raise RuntimeError(f"{what}: dtype must be float32 or bfloat16 (got {dtype})")
    sc = (ctypes.c_float * n)(*_scales(scale, n))
    idc = _check_ids(what, ids)
    V, C = weight.shape
    out = torch.empty(*ids.shape, n, C, dtype=dtype, device=weight.device)
    _launch("mhc_stream_embedding_fwd", weight.device, idc.data_ptr(), ids.dtype == torch.int64, weight.data_ptr(),
            weight.dtype == torch.bfloat16, out.data_ptr(), dtype == torch.bfloat16, sc, idc.numel(), n, C, V)
    return out


def stream_embedding_bwd(grad_out: torch.Tensor, ids: torch.Tensor, num_embeddings: int,
                         scale: Union[float, Sequence[float]] = 1.0, padding_idx: Optional[int] = None,
                         dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """Dense table gradient [num_embeddings, hidden] in ``dtype`` from the
    streams' gradient (ids' shape + [n, hidden]); fp32 sums in a fixed order
    (token order within chunks of sorted tokens, then the chunks' sums)."""
    what = "stream_embedding_bwd"
    _require_cuda(what, grad_out, ids)
    if grad_out.dim() < 2 or grad_out.shape[:-2] != ids.shape:
        raise RuntimeError(f"{what}: grad_out must have ids' shape followed by [n, hidden] "
                           f"(got {tuple(grad_out.shape)} for ids {tuple(ids.shape)})")
    if grad_out.dtype not in _FLOATS or dtype not in _FLOATS:
        raise RuntimeError(f"{what}: grad_out and dtype must be float32 or bfloat16")
    n, C = grad_out.shape[-2:]
    n = _check_n(what, n)
    V = int(num_embeddings)
    pad = _padding(padding_idx, V)
    sc = (ctypes.c_float * n)(*_scales(scale, n))
    idc = _check_ids(what, ids)
    g = grad_out if grad_out.is_contiguous() else grad_out.detach().contiguous()
    gw = torch.empty(V, C, dtype=dtype, device=g.device)
    T = idc.numel()
    ws = _workspace(_lib.mhc_stream_embedding_bwd_workspace_bytes(T, C), g.device)
    _launch("mhc_stream_embedding_bwd", g.device, g.data_ptr(), g.dtype == torch.bfloat16, idc.data_ptr(),
            ids.dtype == torch.int64, gw.data_ptr(), dtype == torch.bfloat16, sc, T, n, C, V, pad, ws.data_ptr(),
            ws.numel())
    return gw


def _padding(padding_idx, V):
    if padding_idx is None:
        return -1
    if not -V <= padding_idx < V:
        raise RuntimeError(f"stream_embedding: padding_idx {padding_idx} is outside a table of {V} rows")
    return padding_idx % V


class StreamEmbeddingFunction(torch.autograd.Function):
    """Embedding lookup into n streams; the table's gradient by sorted tokens."""

    @staticmethod
    def forward(ctx, ids, weight, num_streams, scale, padding_idx, dtype):
        scale = _scales(scale, _check_n("stream_embedding", num_streams))  # the caller's list may change
        out = stream_embedding_fwd(ids, weight.detach(), num_streams, scale, dtype)
        ctx.save_for_backward(ids)
        ctx.args = (weight.size(0), scale, padding_idx, weight.dtype)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_out):
        (ids,) = ctx.saved_tensors
        rows, scale, padding_idx, dtype = ctx.args
        return None, stream_embedding_bwd(grad_out, ids, rows, scale, padding_idx, dtype), None, None, None, None


def stream_embedding(ids: torch.Tensor, weight: torch.Tensor, num_streams: int = 4,
                     scale: Union[float, Sequence[float]] = 1.0, padding_idx: Optional[int] = None,
                     dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """Look token ids up in ``weight`` [vocab, hidden] (float32 or bfloat16) and
    write ``num_streams`` residual streams, stream i scaled by ``scale`` (one
    number, or one for each stream): ids' shape + [n, hidden].  With autograd;
    ``padding_idx``'s row gets no gradient, as in ``torch.nn.Embedding``."""
    if padding_idx is not None and torch.is_tensor(weight) and weight.dim() == 2:
        _padding(padding_idx, weight.size(0))
    return StreamEmbeddingFunction.apply(ids, weight, num_streams, scale, padding_idx, dtype)


class StreamEmbedding(nn.Module):
    """Embedding table whose lookup yields the n residual streams of an mHC
    model (``stream_embedding``)."""

    def __init__(self, num_embeddings: int, hidden_dim: int, num_streams: int = 4,
                 scale: Union[float, Sequence[float]] = 1.0, padding_idx: Optional[int] = None,
                 dtype: Optional[torch.dtype] = None):
        super().__init__()
        self.num_streams, self.scale, self.padding_idx, self.dtype = num_streams, scale, padding_idx, dtype
        self.weight = nn.Parameter(torch.randn(num_embeddings, hidden_dim))
        if padding_idx is not None:
            with torch.no_grad():
                self.weight[_padding(padding_idx, num_embeddings)].zero_()

    def forward(self, ids: torch.Tensor) -> torch.Tensor:
        return stream_embedding(ids, self.weight, self.num_streams, self.scale, self.padding_idx, self.dtype)

    def extra_repr(self) -> str:
        return (f"{self.weight.size(0)}, {self.weight.size(1)}, num_streams={self.num_streams}, "
                f"scale={self.scale}, padding_idx={self.padding_idx}")
