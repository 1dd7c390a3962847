"""Dropout from the counter-based generator, against the generator written again
in unsigned 64-bit integers on the host."""
import ctypes

import numpy as np
import pytest
import torch

import mhc_ascend_b200 as mhc
from mhc_ascend_b200 import _C

F32, BF16 = torch.float32, torch.bfloat16


def philox(counter, key):
    """Philox4x32-10 of counters [n, 4] with one key: [n, 4] words."""
    x = [counter[:, i].astype(np.uint64) for i in range(4)]
    k = [int(key[0]), int(key[1])]
    low, half = np.uint64(0xFFFFFFFF), np.uint64(32)
    for _ in range(10):
        a, b = x[0] * np.uint64(0xD2511F53), x[2] * np.uint64(0xCD9E8D57)
        x = [(b >> half) ^ x[1] ^ np.uint64(k[0]), b & low, (a >> half) ^ x[3] ^ np.uint64(k[1]), a & low]
        k = [(k[0] + 0x9E3779B9) % 2 ** 32, (k[1] + 0xBB67AE85) % 2 ** 32]
    return np.stack(x, 1).astype(np.uint32)


def numbers(seed, position, first, count):
    """16-bit numbers first .. first + count of the stream that starts at `position`."""
    seed %= 2 ** 64
    g0, g1 = first // 8, (first + count + 7) // 8
    groups = [(position + g) % 2 ** 64 for g in range(g0, g1)]
    counter = np.array([(g % 2 ** 32, g >> 32, 0, 0) for g in groups], dtype=np.uint64).reshape(-1, 4)
    w = philox(counter, (seed % 2 ** 32, seed >> 32))
    n = w.reshape(-1).astype("<u4").view("<u2").astype(np.int64)
    return torch.from_numpy(n[first - 8 * g0:first - 8 * g0 + count])


def keep_of(shape, p, rng):
    count = int(np.prod(shape))
    return (numbers(rng[0], rng[1], 0, count) >= round(p * 65536)).view(shape)


def scale_of(p):
    t = round(p * 65536)
    return np.float32(65536.0 / (65536.0 - t)) if t < 65536 else np.float32(0)


def want(x, p, rng):
    """One fp32 product, rounded once."""
    return torch.where(keep_of(x.shape, p, rng), (x.float() * float(scale_of(p))), torch.zeros(())).to(x.dtype)


# ---------------------------------------------------------------------------
# no GPU needed
# ---------------------------------------------------------------------------

def test_published_vectors():
    """Known answers of the generator's authors."""
    f = 0xFFFFFFFF
    for counter, key, words in (
            ((0, 0, 0, 0), (0, 0), (0x6627e8d5, 0xe169c58d, 0xbc57ac4c, 0x9b00dbd8)),
            ((f, f, f, f), (f, f), (0x408f276d, 0x41c83b0e, 0xa20bc7c6, 0x6d5451fd)),
            ((0x243f6a88, 0x85a308d3, 0x13198a2e, 0x03707344), (0xa4093822, 0x299f31d0),
             (0xd16cfe09, 0x94fdcceb, 0x5001e420, 0x24126ea1))):
        assert tuple(philox(np.array([counter], dtype=np.uint64), key)[0]) == words


def test_refusals():
    with pytest.raises(RuntimeError, match="CUDA"):
        mhc.dropout(torch.randn(4), 0.1, (0, 0))
    with pytest.raises(RuntimeError, match="CUDA"):
        mhc.DropoutCounter(3).take(4)
    with pytest.raises(RuntimeError, match=r"p must be in \[0, 1\]"):
        mhc.StreamDropout(1.5)
    with pytest.raises(RuntimeError, match=r"p must be in \[0, 1\]"):
        mhc.StreamDropout(float("nan"))
    assert mhc.dropout_groups((3, 5)) == 2 and mhc.dropout_groups((0, 5)) == 0


def test_counter_state_is_saved():
    a = mhc.DropoutCounter(seed=2 ** 64 - 5, position=7)
    assert a.state.tolist() == [-5, 7]
    b = mhc.DropoutCounter()
    b.load_state_dict(a.state_dict())
    assert b.state.tolist() == [-5, 7]
    layer = mhc.StreamDropout(0.3, seed=4)
    assert layer.eval()(torch.ones(3)).tolist() == [1, 1, 1] and list(layer.state_dict()) == ["counter.state"]
    assert layer.half().counter.state.dtype == torch.int64


def test_entry_points_validate_without_gpu():
    lib = _C.load()
    p, odd = ctypes.c_void_p(16), ctypes.c_void_p(20)
    assert lib.mhc_dropout(p, 0, p, 0, 10, None, 0, 0, None) == 0
    assert lib.mhc_dropout(p, 0, p, -1, 10, None, 0, 0, None) == -1
    assert lib.mhc_dropout(p, 0, p, 8, 65537, None, 0, 0, None) == -1 and "65536" in _C.last_error()
    assert lib.mhc_dropout(p, 0, p, 8, -1, None, 0, 0, None) == -1
    assert lib.mhc_dropout(None, 0, p, 8, 1, None, 0, 0, None) == -1
    assert lib.mhc_dropout(p, 0, None, 8, 1, None, 0, 0, None) == -1
    assert lib.mhc_dropout(p, 0, p, 8, 1, odd, 0, 0, None) == -3
    assert lib.mhc_dropout_take(None, p, 8, None) == -1 and lib.mhc_dropout_take(p, p, -1, None) == -1
    assert lib.mhc_dropout_take(p, odd, 8, None) == -3


# ---------------------------------------------------------------------------
# GPU
# ---------------------------------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("count", [0, 1, 7, 8, 9, 255, 256, 4099, 4096, 8192, 100003])
def test_values(cuda, count, dtype):
    gen = torch.Generator().manual_seed(count)
    x = torch.randn(count, generator=gen).to(dtype)
    for p, rng in ((0.1, (count, 5)), (0.5, (-3, 2 ** 32 - 2)), (1e-6, (7, 0)), (0.0, (7, 0)), (1.0, (1, 1))):
        got = mhc.dropout(x.to(cuda), p, rng)
        assert got.dtype == dtype and torch.equal(got.cpu(), want(x, p, rng))


@pytest.mark.gpu
@pytest.mark.parametrize("rng", [(0, 0), (2 ** 64 - 1, 2 ** 64 - 3), (1 << 40, (5 << 32) - 1)])
def test_seeds_and_positions_of_64_bits(cuda, rng):
    x = torch.randn(100, generator=torch.Generator().manual_seed(1))
    assert torch.equal(mhc.dropout_fwd(x.to(cuda), 0.4, rng).cpu(), want(x, 0.4, rng))
    words = torch.tensor([v - 2 ** 64 if v >> 63 else v for v in rng], device=cuda)
    assert torch.equal(mhc.dropout_fwd(x.to(cuda), 0.4, words).cpu(), want(x, 0.4, rng))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_layouts(cuda, dtype):
    """Starts that are not aligned, and tensors that are not contiguous."""
    base = torch.randn(1000, device=cuda).to(dtype)
    for off in (1, 2, 3, 5, 8):
        x = base[off:off + 900]
        assert torch.equal(mhc.dropout(x, 0.3, (9, 9)).cpu(), want(x.cpu(), 0.3, (9, 9)))
    x = base[:960].view(30, 32)
    for v in (x.t(), x[:, 3:20], x[::2], x[:1].expand(30, 32), x.view(2, 15, 32).transpose(0, 1)):
        got = mhc.dropout(v, 0.3, (9, 9))
        assert got.is_contiguous() and torch.equal(got.cpu(), want(v.cpu(), 0.3, (9, 9)))
    scalar = torch.tensor(2.0, device=cuda, dtype=dtype)
    assert mhc.dropout(scalar, 0.0, (1, 1)).item() == 2.0


@pytest.mark.gpu
def test_infinities_and_nans_are_dropped(cuda):
    x = torch.full((64,), float("nan"))
    x[::2] = float("inf")
    keep = keep_of((64,), 0.5, (3, 3))
    got = mhc.dropout(x.to(cuda), 0.5, (3, 3)).cpu()
    assert not got[~keep].any() and torch.equal(torch.isnan(got), keep & torch.isnan(x))


@pytest.mark.gpu
def test_more_values_than_32_bits_count(cuda):
    count, rng = 2 ** 32 + 2 ** 12 + 5, (11, 2 ** 33)
    x = torch.ones(count, device=cuda, dtype=BF16)
    got = mhc.dropout_fwd(x, 0.25, rng)
    for first in (0, 2 ** 31 - 50, 2 ** 32 - 50, count - 101):
        keep = numbers(*rng, first, 100) >= 16384
        assert torch.equal(got[first:first + 100].cpu() != 0, keep)
    share = (got != 0).sum().item() / count
    assert abs(share - 0.75) < 6 * (0.75 * 0.25 / count) ** 0.5


@pytest.mark.gpu
def test_gradient(cuda):
    x = torch.randn(50, 37, device=cuda, requires_grad=True)
    g = torch.randn(50, 37, device=cuda)
    out = mhc.dropout(x, 0.2, (5, 6))
    out.backward(g)
    assert torch.equal(x.grad.cpu(), want(g.cpu(), 0.2, (5, 6)))
    # the function is linear: differences give the gradient's product with a direction
    d = torch.randn(50, 37, device=cuda)
    up, down = (mhc.dropout_fwd((x.detach() + s * d), 0.2, (5, 6)).double() for s in (1, -1))
    slope = ((up - down) / 2 * g.double()).sum().item()
    # products and sums of 1850 values of size ~1, each rounded at 2^-24 a few times
    assert slope == pytest.approx((x.grad.double() * d.double()).sum().item(), abs=1850 * 8 * 2.0 ** -24 * 4)
    with pytest.raises(RuntimeError):  # not differentiable again
        y = mhc.dropout(x, 0.2, (5, 6))
        (gx,) = torch.autograd.grad((y * y).sum(), x, create_graph=True)
        gx.sum().backward()


@pytest.mark.gpu
def test_counter(cuda):
    c = mhc.DropoutCounter(seed=9, position=2 ** 33).to(cuda)
    a, b = c.take(10), c.take(0)
    assert a.tolist() == [9, 2 ** 33] and b.tolist() == [9, 2 ** 33 + 10] and c.state.tolist() == [9, 2 ** 33 + 10]
    layer = mhc.StreamDropout(0.3, seed=9).to(cuda)
    x = torch.ones(3, 50, device=cuda, requires_grad=True)
    first, second = layer(x), layer(x)
    assert torch.equal(first.detach().cpu(), want(torch.ones(3, 50), 0.3, (9, 0)))
    assert torch.equal(second.detach().cpu(), want(torch.ones(3, 50), 0.3, (9, mhc.dropout_groups((3, 50)))))
    first.sum().backward()  # after the counter has moved on
    assert torch.equal(x.grad, first.detach())
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    taken = []
    for i in range(60):
        with torch.cuda.stream(streams[i % 3]):
            taken.append(c.take(5))
    torch.cuda.synchronize()
    assert sorted(t[1].item() for t in taken) == [2 ** 33 + 10 + 5 * i for i in range(60)]


@pytest.mark.gpu
def test_captured_graph_draws_new_masks(cuda):
    layer = mhc.StreamDropout(0.4, seed=2).to(cuda)
    x = torch.randn(33, 40, device=cuda, requires_grad=True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        layer(x).sum().backward()
    torch.cuda.current_stream().wait_stream(side)
    x.grad = None
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = layer(x)
        (gx,) = torch.autograd.grad(out.sum(), x)
    groups = mhc.dropout_groups(x.shape)
    for turn in range(3):
        graph.replay()
        rng = (2, (1 + turn) * groups)
        assert torch.equal(out.detach().cpu(), want(x.detach().cpu(), 0.4, rng))
        assert torch.equal(gx.cpu(), want(torch.ones(33, 40), 0.4, rng))


@pytest.mark.gpu
def test_recomputation_draws_the_same_mask(cuda):
    """What a function that runs twice may draw: numbers at a given position."""
    x = torch.randn(20, 4, 64, device=cuda, requires_grad=True)
    out = mhc.checkpoint8_recompute(lambda t: mhc.dropout(t * t, 0.3, (1, 2)), x)
    assert torch.equal(out, mhc.dropout(x * x, 0.3, (1, 2)))
    out.sum().backward()
    restored = mhc.checkpoint8_pack(x.detach()).unpack()
    scaled = want(torch.ones(20, 4, 64), 0.3, (1, 2)).to(cuda)
    assert torch.equal(x.grad, scaled * restored + scaled * restored)


@pytest.mark.gpu
def test_recomputation_takes_no_new_numbers(cuda):
    """A counter inside would draw another mask when the function runs again."""
    layer = mhc.StreamDropout(0.3).to(cuda)
    x = torch.randn(4, 64, device=cuda, requires_grad=True)
    with pytest.raises(RuntimeError, match="may not take new numbers"):
        mhc.checkpoint8_recompute(layer, x)
    assert layer.counter.state.tolist() == [0, 0]
    with torch.no_grad():  # runs once
        mhc.checkpoint8_recompute(layer, x)
    rng = layer.counter.take(mhc.dropout_groups(x.shape))
    out = mhc.checkpoint8_recompute(lambda t: mhc.dropout(t, layer.p, rng), x)
    out.sum().backward()
    assert torch.equal(x.grad != 0, out != 0)
    assert torch.equal(layer(x.detach()) != 0, mhc.dropout(x.detach(), 0.3, (0, 64)) != 0)  # and is free again


@pytest.mark.gpu
def test_gpu_refusals(cuda):
    x = torch.randn(8, device=cuda)
    for rng in (5, (1, 2, 3), "ab", torch.zeros(2, device=cuda), torch.zeros(3, dtype=torch.int64, device=cuda)):
        with pytest.raises(RuntimeError, match="rng"):
            mhc.dropout(x, 0.1, rng)
    with pytest.raises(RuntimeError, match="rng must be on"):
        mhc.dropout(x, 0.1, torch.zeros(2, dtype=torch.int64))
    with pytest.raises(RuntimeError, match="float32 or bfloat16"):
        mhc.dropout(x.half(), 0.1, (0, 0))
    with pytest.raises(RuntimeError, match="p must be"):
        mhc.dropout(x, -0.1, (0, 0))
    rng = torch.tensor([1, 2], device=cuda)
    y = mhc.dropout(x.requires_grad_(True), 0.5, rng)
    rng[1] += 1  # the backward pass would draw another mask
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
