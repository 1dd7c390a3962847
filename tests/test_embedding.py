"""Embedding lookup into streams and its gradient, against 64-bit sums."""
import pytest
import torch

import mhc_ascend_b200 as mhc
from mhc_ascend_b200 import _C

U = 2.0 ** -24  # unit roundoff of fp32
UB = 2.0 ** -8  # of bf16: 8 significant bits against 24
F32, BF16 = torch.float32, torch.bfloat16


# ---------------------------------------------------------------------------
# refusals (no GPU needed)
# ---------------------------------------------------------------------------

def test_cpu_tensors_raise():
    with pytest.raises(RuntimeError, match="CUDA"):
        mhc.stream_embedding(torch.zeros(3, dtype=torch.int64), torch.randn(4, 8))
    with pytest.raises(RuntimeError, match="CUDA"):
        mhc.stream_embedding_bwd(torch.randn(3, 4, 8), torch.zeros(3, dtype=torch.int64), 4)


def test_padding_outside_the_table_raises():
    with pytest.raises(RuntimeError, match="padding_idx"):
        mhc.stream_embedding(torch.zeros(3, dtype=torch.int64), torch.randn(4, 8), padding_idx=4)
    with pytest.raises(RuntimeError, match="padding_idx"):
        mhc.StreamEmbedding(4, 8, padding_idx=-5)


def test_entry_points_validate_without_gpu():
    lib = _C.load()
    import ctypes
    p, odd = ctypes.c_void_p(16), ctypes.c_void_p(20)
    sc = (ctypes.c_float * 32)(*([1.0] * 32))

    def fwd(ids=p, w=p, out=p, s=sc, T=4, n=4, C=8, V=16):
        return lib.mhc_stream_embedding_fwd(ids, 1, w, 0, out, 0, s, T, n, C, V, None)

    def bwd(g=p, ids=p, gw=p, s=sc, T=4, n=4, C=8, V=16, ws=p, size=1 << 30):
        return lib.mhc_stream_embedding_bwd(g, 0, ids, 1, gw, 0, s, T, n, C, V, -1, ws, size, None)

    assert fwd(T=0) == 0
    assert fwd(n=0) == -2 and fwd(n=33) == -2 and "[1, 32]" in _C.last_error()
    assert fwd(T=-1) == -1 and fwd(C=0) == -1 and fwd(V=0) == -1
    assert fwd(ids=None) == -1 and fwd(w=None) == -1 and fwd(out=None) == -1 and fwd(s=None) == -1
    assert fwd(T=1 << 31) == -2 and fwd(V=1 << 31) == -2
    assert bwd(n=33) == -2 and bwd(V=0) == -1 and bwd(g=None) == -1 and bwd(gw=None) == -1
    assert bwd(gw=odd) == -3
    assert bwd(ws=None) == -4 and bwd(size=16) == -4
    assert lib.mhc_stream_embedding_bwd_workspace_bytes(-1, 8) == 0


# ---------------------------------------------------------------------------
# GPU
# ---------------------------------------------------------------------------

def _ids(T, V, kind, gen, dtype=torch.int64):
    if kind == "same":
        ids = torch.full((T,), V // 2)
    elif kind == "distinct":
        ids = torch.randperm(max(T, V), generator=gen)[:T] % V
    elif kind == "falling":
        ids = torch.arange(T).flip(0) % V
    else:  # frequency ~ 1 / rank
        ids = (torch.exp(torch.rand(T, generator=gen) * torch.log(torch.tensor(float(V)))).long() - 1).clamp_(0, V - 1)
    return ids.to(dtype)


def _grad64(g, ids, V, scales, pad=None):
    """(gradient, sum of |terms|, terms per row) in 64 bits."""
    keep = (ids >= 0) & (ids < V)
    if pad is not None:
        keep &= ids != pad
    s = torch.tensor(scales).double()[None, :, None]
    terms = g.double()[keep] * s
    out, mag = (torch.zeros(V, g.size(-1), dtype=torch.float64) for _ in range(2))
    out.index_add_(0, ids[keep].long(), terms.sum(1))
    mag.index_add_(0, ids[keep].long(), terms.abs().sum(1))
    count = torch.bincount(ids[keep].long(), minlength=V).double() * g.size(1)
    return out, mag, count


def _check_grad(got, want, mag, count, bf16):
    # each of a row's `count` additions (and the joins of its parts, fewer) rounds
    # a partial sum that is at most `mag`
    tol = 2 * count[:, None] * U * mag + (UB * want.abs() * (1 + UB) if bf16 else 0)
    err = (got.double().cpu() - want).abs()
    assert bool((err <= tol).all()), f"max excess {(err - tol).max():.3g}"


@pytest.mark.gpu
@pytest.mark.parametrize("T,n,C,V", [(1, 4, 8, 2), (7, 1, 1, 5), (33, 3, 31, 100), (257, 4, 256, 1000),
                                     (64, 32, 1280, 300), (5, 2, 4099, 7), (3000, 1, 4, 70000)])
@pytest.mark.parametrize("tw,to", [(F32, F32), (F32, BF16), (BF16, F32), (BF16, BF16)])
def test_forward(cuda, T, n, C, V, tw, to):
    gen = torch.Generator().manual_seed(T * 7 + C)
    w = torch.randn(V, C, generator=gen).to(tw)
    ids = _ids(T, V, "text", gen, torch.int32 if n % 2 else torch.int64)
    scales = [0.3 + 0.7 * i for i in range(n)]
    out = mhc.stream_embedding(ids.to(cuda), w.to(cuda), n, scales, dtype=to)
    want = (w[ids.long()].float()[:, None] * torch.tensor(scales)[None, :, None]).to(to)
    assert out.dtype == to and torch.equal(out.cpu(), want)  # one fp32 product, rounded once


@pytest.mark.gpu
def test_forward_shapes_scale_and_bad_ids(cuda):
    w = torch.randn(10, 16, device=cuda)
    ids = torch.tensor([[0, 9, 10], [-1, 3, 1 << 40]], device=cuda)
    out = mhc.stream_embedding(ids, w, 2, 0.5)
    assert out.shape == (2, 3, 2, 16)
    bad = torch.tensor([[False, False, True], [True, False, True]])
    assert torch.equal(torch.isnan(out).all(-1).all(-1).cpu(), bad)
    assert torch.equal(out[0, 1, 1], w[9] * 0.5) and torch.equal(out[1, 1, 0], w[3] * 0.5)
    assert mhc.stream_embedding(ids[:0], w, 3).shape == (0, 3, 3, 16)
    one = mhc.stream_embedding(torch.tensor(4, device=cuda), w, 1)
    assert one.shape == (1, 16) and torch.equal(one[0], w[4])


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["text", "same", "distinct", "falling"])
@pytest.mark.parametrize("T,n,C,V", [(1, 4, 8, 1), (2, 1, 3, 2), (31, 2, 5, 9), (32, 4, 64, 40), (33, 3, 36, 511),
                                     (64, 1, 129, 512), (65, 2, 132, 513), (2047, 1, 12, 300),
                                     (2049, 2, 4, 70000), (16385, 1, 4, 1000), (40000, 1, 3, 262200)])
def test_gradient_sizes(cuda, T, n, C, V, kind):
    gen = torch.Generator().manual_seed(T + V)
    g = torch.randn(T, n, C, generator=gen)
    ids = _ids(T, V, kind, gen)
    scales = [1.5 - 0.4 * i for i in range(n)]
    got = mhc.stream_embedding_bwd(g.to(cuda), ids.to(cuda), V, scales)
    _check_grad(got, *_grad64(g, ids, V, scales), bf16=False)
    assert torch.equal(got, mhc.stream_embedding_bwd(g.to(cuda), ids.to(cuda), V, scales))  # bitwise


@pytest.mark.gpu
@pytest.mark.parametrize("tg,tw", [(F32, BF16), (BF16, F32), (BF16, BF16)])
@pytest.mark.parametrize("C", [64, 65])
def test_gradient_types(cuda, tg, tw, C):
    gen = torch.Generator().manual_seed(C)
    T, n, V = 700, 4, 90
    g, ids = torch.randn(T, n, C, generator=gen).to(tg), _ids(T, V, "text", gen, torch.int32)
    got = mhc.stream_embedding_bwd(g.to(cuda), ids.to(cuda), V, 0.7, dtype=tw)
    assert got.dtype == tw
    _check_grad(got, *_grad64(g, ids, V, [0.7] * n), bf16=tw == BF16)


@pytest.mark.gpu
@pytest.mark.parametrize("pad", [0, 5, -1])
def test_gradient_padding_and_bad_ids(cuda, pad):
    gen = torch.Generator().manual_seed(pad + 3)
    T, n, C, V = 500, 2, 20, 33
    ids = _ids(T, V, "text", gen)
    ids[::3] = pad % V
    ids[1::7] = -100
    ids[2::11] = V
    g = torch.randn(T, n, C, generator=gen)
    got = mhc.stream_embedding_bwd(g.to(cuda), ids.to(cuda), V, 1.0, padding_idx=pad)
    _check_grad(got, *_grad64(g, ids, V, [1.0] * n, pad % V), bf16=False)
    assert not got[pad % V].any()
    every = torch.full((T,), pad % V)  # nothing but padding
    assert not mhc.stream_embedding_bwd(g.to(cuda), every.to(cuda), V, 1.0, padding_idx=pad).any()


@pytest.mark.gpu
def test_gradient_of_nothing_and_of_nan(cuda):
    g = torch.randn(0, 3, 8, device=cuda)
    none = torch.zeros(0, dtype=torch.int64, device=cuda)
    assert not mhc.stream_embedding_bwd(g, none, 6).any()
    g = torch.ones(4, 1, 8, device=cuda)
    g[2, 0, 3] = float("inf")
    g[3, 0, 4] = float("nan")
    gw = mhc.stream_embedding_bwd(g, torch.tensor([0, 1, 2, 3], device=cuda), 5)
    assert torch.isinf(gw[2, 3]) and torch.isnan(gw[3, 4]) and int(torch.isfinite(gw).sum()) == 5 * 8 - 2


@pytest.mark.gpu
def test_autograd_layouts_and_streams(cuda):
    """Expanded and transposed gradients, unaligned storage, a side stream."""
    gen = torch.Generator().manual_seed(1)
    V, C, T, n = 50, 24, 60, 3
    w0 = torch.randn(V, C, generator=gen)
    ids = _ids(T, V, "text", gen)
    layer = mhc.StreamEmbedding(V, C, n, [1.0, 0.5, 0.25], padding_idx=2).to(cuda)
    assert not layer.weight[2].any()
    with torch.no_grad():
        layer.weight.copy_(w0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        layer(ids.to(cuda)).sum().backward()  # the gradient is an expanded scalar
    torch.cuda.current_stream().wait_stream(side)
    ones = torch.ones(T, n, C)
    _check_grad(layer.weight.grad, *_grad64(ones, ids, V, [1.0, 0.5, 0.25], 2), bf16=False)
    store = torch.randn(T * n * C + 1, generator=gen).to(cuda)
    g = store[1:].view(T, n, C)  # 4-byte aligned only
    got = mhc.stream_embedding_bwd(g, ids.to(cuda), V)
    _check_grad(got, *_grad64(g.cpu(), ids, V, [1.0] * n), bf16=False)
    gt = torch.randn(C, n, T, generator=gen).to(cuda).permute(2, 1, 0)
    got = mhc.stream_embedding_bwd(gt, ids.to(cuda)[::1], V)
    _check_grad(got, *_grad64(gt.cpu(), ids, V, [1.0] * n), bf16=False)


@pytest.mark.gpu
def test_gradient_against_differences(cuda):
    """The lookup is linear in the table: a difference is the derivative."""
    gen = torch.Generator().manual_seed(9)
    V, C, T, n = 40, 32, 100, 4
    ids = _ids(T, V, "text", gen).to(cuda)
    w = torch.randn(V, C, generator=gen).to(cuda).requires_grad_(True)
    g = torch.randn(T, n, C, generator=gen).to(cuda)
    scales = [2.0, 1.0, 0.5, 0.25]
    mhc.stream_embedding(ids, w, n, scales).backward(g)
    v = torch.randn(V, C, generator=gen).to(cuda)
    with torch.no_grad():
        up, down = (mhc.stream_embedding(ids, w + h * v, n, scales).double() for h in (0.5, -0.5))
    slope = ((up - down) * g.double()).sum()
    # products and table sums round at U of their size, of random sign over T n C values
    size = ((up.abs() + down.abs()) * g.double().abs()).norm() + (w.grad.double() * v.double()).norm() * 4 * n
    assert abs(slope - (w.grad.double() * v.double()).sum()) <= 8 * U * size


@pytest.mark.gpu
def test_refusals(cuda):
    w = torch.randn(8, 16, device=cuda)
    ids = torch.zeros(3, dtype=torch.int64, device=cuda)
    with pytest.raises(RuntimeError, match="num_streams"):
        mhc.stream_embedding(ids, w, 33)
    with pytest.raises(RuntimeError, match="scales"):
        mhc.stream_embedding(ids, w, 4, [1.0, 2.0])
    with pytest.raises(RuntimeError, match="int64 or int32"):
        mhc.stream_embedding(ids.float(), w, 4)
    with pytest.raises(RuntimeError, match="contiguous"):
        mhc.stream_embedding(ids, w.t(), 4)
    with pytest.raises(RuntimeError, match="float32 or bfloat16"):
        mhc.stream_embedding(ids, w, 4, dtype=torch.float16)
    with pytest.raises(RuntimeError, match="ids' shape"):
        mhc.stream_embedding_bwd(torch.randn(4, 2, 16, device=cuda), ids, 8)


@pytest.mark.gpu
def test_offsets_past_32_bits(cuda):
    """Streams and tables of more than 2^31 values."""
    T, n, C, V = 70000, 8, 4096, 600
    w = torch.randn(V, C, device=cuda, dtype=BF16)
    ids = torch.randint(0, V, (T,), device=cuda)
    out = mhc.stream_embedding(ids, w, n)
    for t in (0, T // 2, T - 1):
        assert torch.equal(out[t, n - 1], w[ids[t]])
    del out
    V = 530000
    ids = torch.tensor([0, 3, V - 1, V - 2, V - 1], device=cuda)
    g = torch.ones(5, 1, C, device=cuda, dtype=BF16)
    gw = mhc.stream_embedding_bwd(g, ids, V, dtype=BF16)
    assert float(gw[V - 1].float().sum()) == 2 * C and float(gw[V - 2].float().sum()) == C
    assert float(gw.sum(dtype=torch.float32)) == 5 * C


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [list, torch.tensor])
def test_gradient_uses_the_forwards_scales(cuda, kind):
    """Scales that change after the lookup change nothing in its gradient."""
    scales = kind([1.0, 0.5])
    w = torch.randn(6, 8, device=cuda, requires_grad=True)
    out = mhc.stream_embedding(torch.tensor([1, 4], device=cuda), w, 2, scales)
    scales[0] = 100.0
    out.sum().backward()
    assert torch.equal(w.grad.sum(1).cpu(), torch.tensor([0.0, 12.0, 0.0, 0.0, 12.0, 0.0]))


@pytest.mark.gpu
@pytest.mark.parametrize("T", [30000, 70000])  # 32 and 64 positions a block
@pytest.mark.parametrize("kind,pad", [("text", None), ("text", 0), ("same", None)])
@pytest.mark.parametrize("tg,tw,C,shift", [(BF16, BF16, 1281, 0), (BF16, F32, 1281, 1), (BF16, BF16, 1280, 0),
                                           (BF16, F32, 1280, 1), (F32, F32, 1281, 0), (F32, BF16, 1284, 0),
                                           (F32, F32, 1284, 1)])
def test_gradient_of_training_batches(cuda, T, kind, pad, tg, tw, C, shift):
    """Blocks of many positions and rows of several slices, in the layouts that
    16-byte accesses fit and in those that they do not (an odd width; a start
    that is `shift` values off)."""
    n, V, scales = 2, 5000, [1.0, -0.625]
    cpu = torch.Generator().manual_seed(T + C)
    gen = torch.Generator(device=cuda).manual_seed(T + C)
    ids = _ids(T, V, kind, cpu)
    if pad is not None:
        ids[torch.rand(T, generator=cpu) < 0.2] = pad
    ids = ids.to(cuda)
    store = torch.randn(T * n * C + shift, device=cuda, generator=gen).to(tg)
    g = store[shift:].view(T, n, C)
    got = mhc.stream_embedding_bwd(g, ids, V, scales, padding_idx=pad, dtype=tw)
    want, mag = (torch.zeros(V, C, dtype=torch.float64, device=cuda) for _ in range(2))
    keep = torch.arange(T, device=cuda) if pad is None else torch.nonzero(ids != pad).squeeze(1)
    for i, s in enumerate(scales):
        term = g[:, i].double()[keep] * s
        want.index_add_(0, ids[keep], term)
        mag.index_add_(0, ids[keep], term.abs())
    count = torch.bincount(ids[keep], minlength=V).double() * n
    bf16 = tw == BF16
    _check_grad(got, want.cpu(), mag.cpu(), count.cpu(), bf16)
    # over the whole table: a row's roundings are of random sign
    err = (got.double() - want).norm()
    bound = ((count.sqrt() + 8)[:, None] * U * mag).norm() + (UB * (1 + UB) * want.norm() if bf16 else 0)
    assert float(err) <= float(bound)
    assert torch.equal(got, mhc.stream_embedding_bwd(g, ids, V, scales, padding_idx=pad, dtype=tw))
