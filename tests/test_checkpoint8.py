"""8-bit checkpoints: the format, and the backward operators that read it,
against 64-bit formulas at the restored input."""
import ctypes

import pytest
import torch

import mhc_ascend_b200 as mhc
from mhc_ascend_b200 import _C

U = 2.0 ** -24  # unit roundoff of fp32
UB = 2.0 ** -8  # of bf16: 8 significant bits against 24
F32, BF16 = torch.float32, torch.bfloat16


def restored64(x):
    """What x stands for after 8 bits, by the definition, in 64 bits on the CPU."""
    x = x.detach().double().cpu()
    cols = x.size(-1)
    n = -(-cols // 32)
    f = torch.zeros(x.numel() // cols, n * 32, dtype=torch.float64)
    f[:, :cols] = x.reshape(-1, cols)
    f = f.view(-1, n, 32)
    a = f.abs().amax(-1)
    m, e = torch.frexp(a)
    e = torch.where(m < 127.5 / 128, e - 7, e - 6).clamp(min=-126)
    step = torch.exp2(e.double()).unsqueeze(-1)  # exact on the CPU for whole e
    out = torch.round(f / step) * step
    # 64 steps of 2^122 would be 2^128, past fp32: 63 of them are the most
    out = torch.where(out.abs() >= 2.0 ** 128, out.sign() * 63 * 2.0 ** 122, out)
    out = torch.where(torch.isfinite(a).unsqueeze(-1), out, torch.full_like(out, float("nan")))
    return out.view(-1, n * 32)[:, :cols].reshape(x.shape)


def acts(*shape, seed=0, dtype=F32):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(*shape, generator=gen) * torch.exp(torch.randn(shape[-1], generator=gen))
    return x.to(dtype)


# ---------------------------------------------------------------------------
# refusals (no GPU needed)
# ---------------------------------------------------------------------------

def test_cpu_tensors_raise():
    for call in (lambda: mhc.checkpoint8_pack(torch.randn(4, 8)),
                 lambda: mhc.rmsnorm_checkpoint8(torch.randn(4, 8), torch.ones(8)),
                 lambda: mhc.linear_checkpoint8(torch.randn(4, 8), torch.randn(3, 8)),
                 lambda: mhc.Checkpoint8(torch.zeros(2, 128, dtype=torch.int8), torch.zeros(2, 4, dtype=torch.uint8),
                                         (2, 8), F32)):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()
    with pytest.raises(RuntimeError, match="kept"):
        mhc.checkpoint8_recompute(lambda t: t, torch.randn(2, 2), kept=2)


def test_entry_points_validate_without_gpu():
    lib = _C.load()
    p, odd = ctypes.c_void_p(16), ctypes.c_void_p(18)
    assert [lib.mhc_checkpoint8_pitch(c) for c in (0, 1, 128, 129)] == [0, 128, 128, 256]
    pack = lambda x=p, st=8, c=p, e=p, r=4, n=8: lib.mhc_checkpoint8_pack(x, 0, st, c, e, r, n, None)  # noqa: E731
    assert pack(r=0) == 0 and pack(r=-1) == -1 and pack(n=0) == -1 and pack(x=None) == -1
    assert pack(st=7) == -1 and "row_stride" in _C.last_error()
    assert pack(c=None) == -1 and pack(c=odd) == -3 and pack(e=odd) == -3
    assert pack(r=1 << 40, n=1 << 20) == -2
    un = lambda c=p, e=p, o=p, r=4, n=8: lib.mhc_checkpoint8_unpack(c, e, o, 0, r, n, None)  # noqa: E731
    assert un(r=0) == 0 and un(o=None) == -1 and un(c=odd) == -3 and un(n=0) == -1
    fwd = lambda eps=1e-5, w=p, rms=p: lib.mhc_rmsnorm_checkpoint8_fwd(  # noqa: E731
        p, 0, w, p, rms, p, p, 4, 8, eps, None)
    assert fwd(eps=-1.0) == -1 and fwd(w=None) == -1 and fwd(rms=None) == -1
    bwd = lambda ws=p, size=1 << 20, gw=p: lib.mhc_rmsnorm_checkpoint8_bwd(  # noqa: E731
        p, 0, p, p, p, p, p, gw, 4, 8, ws, size, None)
    assert bwd(ws=None) == -4 and bwd(size=1) == -4 and bwd(gw=None) == -1
    wg = lambda g=p, st=8, c=p, gw=p, T=4, O=8, K=8: lib.mhc_checkpoint8_weight_grad(  # noqa: E731
        g, 1, st, c, p, gw, 0, T, O, K, None, 0, None)
    assert wg(T=-1) == -1 and wg(O=0) == -1 and wg(K=0) == -1 and wg(g=None) == -1 and wg(gw=None) == -1
    assert wg(st=7) == -1 and wg(c=odd) == -3 and wg(T=1 << 31) == -2
    size = lambda *a: lib.mhc_checkpoint8_weight_grad_workspace_bytes(*a)  # noqa: E731
    assert size(-1, 8, 8, 1, 1) == 0 and size(100, 8, 8, 1, 0) - size(100, 8, 8, 1, 1) >= 1600
    assert wg(g=ctypes.c_void_p(18)) == -4 and "workspace" in _C.last_error()  # needs a copy


# ---------------------------------------------------------------------------
# format
# ---------------------------------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 31), (2, 32), (5, 33), (7, 127), (4, 128), (9, 129), (64, 8),
                                       (1, 4097), (33, 1280), (300, 264)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_pack_restores_the_definition(cuda, rows, cols, dtype):
    x = acts(rows, cols, seed=cols, dtype=dtype)
    kept = mhc.checkpoint8_pack(x.to(cuda))
    want = restored64(x)
    assert kept.codes.shape == (rows, -(-cols // 128) * 128) and int(kept.codes.min()) >= -127
    for t in (F32, BF16):  # 8 significant bits: exact in both
        got = kept.unpack(t)
        assert got.dtype == t and torch.equal(got.double().cpu(), want)
    again = mhc.checkpoint8_pack(kept.unpack())
    assert torch.equal(again.unpack(), kept.unpack())  # what is restored packs to itself
    # code k of block b is k * 2^(E - 127), padding is zero
    step = torch.exp2(kept.exponents.double().cpu() - 127).repeat_interleave(32, 1)
    values = kept.codes.double().cpu() * step
    assert torch.equal(values[:, :cols], want) and not values[:, cols:].any()


@pytest.mark.gpu
def test_pack_edges(cuda):
    rows = [
        [127.5, -127.49999, 126.5, 125.5, 0.5, 1.5, -0.5, 2.5],  # the threshold takes the next step; ties to even
        [127.49999, 126.5, -126.5, 0.5, -1.5, 0.49999997, 0.0, -0.0],
        [3.4e38, -3.4e38, 1.0, 2.0 ** 121, 2.0 ** 122, 0, 0, 0],  # the largest finite values
        [2.0 ** -126, 2.0 ** -127, 2.0 ** -149, -(2.0 ** -126) * 1.5, 0, 0, 0, 0],  # subnormals round to the smallest step
        [0.0] * 8,
    ]
    x = torch.zeros(len(rows), 32)
    x[:, :8] = torch.tensor(rows)
    for xx in (x, torch.cat([x, x * 2.0 ** -3, x], 1), x[:, :8].contiguous()):
        assert torch.equal(mhc.checkpoint8_pack(xx.to(cuda)).unpack().double().cpu(), restored64(xx))
    every = torch.arange(-127, 128).float() * 2.0 ** -5  # every code
    x = torch.stack([torch.roll(every, k) for k in range(32)])
    x[:, ::32] = 127 * 2.0 ** -5
    assert torch.equal(mhc.checkpoint8_pack(x.to(cuda)).unpack().cpu(), x)


@pytest.mark.gpu
@pytest.mark.parametrize("bad", [float("inf"), -float("inf"), float("nan")])
@pytest.mark.parametrize("cols", [96, 97])
def test_block_with_a_bad_value_is_nan(cuda, bad, cols):
    x = acts(6, cols, seed=3)
    x[2, 40] = bad
    x[5, 0] = bad
    got = mhc.checkpoint8_pack(x.to(cuda)).unpack().cpu()
    want = restored64(x)
    assert torch.equal(torch.isnan(got), torch.isnan(want)) and int(torch.isnan(got).sum()) == 64
    assert torch.equal(torch.nan_to_num(got.double()), torch.nan_to_num(want))


@pytest.mark.gpu
def test_pack_layouts(cuda):
    base = acts(20, 3 * 64, seed=4).to(cuda)
    cut = base[:, 64:128]  # strided rows, aligned
    assert torch.equal(mhc.checkpoint8_pack(cut).unpack().double().cpu(), restored64(cut))
    cut = base[1:, 3:100]  # strided rows, unaligned
    assert torch.equal(mhc.checkpoint8_pack(cut).unpack().double().cpu(), restored64(cut))
    flip = base.t()
    kept = mhc.checkpoint8_pack(flip)
    assert kept.shape == flip.shape and torch.equal(kept.unpack().double().cpu(), restored64(flip))
    deep = acts(2, 3, 5, 40, seed=5).to(cuda)
    assert torch.equal(mhc.checkpoint8_pack(deep).unpack().double().cpu(), restored64(deep))
    wide = deep[:, :1].expand(2, 3, 5, 40)
    assert torch.equal(mhc.checkpoint8_pack(wide).unpack().double().cpu(), restored64(wide))
    flat = deep.reshape(-1)
    assert torch.equal(mhc.checkpoint8_pack(flat).unpack().double().cpu(), restored64(flat))
    none = mhc.checkpoint8_pack(deep[:0])
    assert none.unpack().shape == (0, 3, 5, 40)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = mhc.checkpoint8_pack(deep).unpack()
    side.synchronize()
    assert torch.equal(got.double().cpu(), restored64(deep))


@pytest.mark.gpu
def test_pack_past_32_bits(cuda):
    rows, cols = 525000, 4096  # 2.15e9 values
    x = torch.empty(rows, cols, dtype=BF16, device=cuda).normal_()
    kept = mhc.checkpoint8_pack(x)
    back = kept.unpack()
    for r in (0, rows // 2, rows - 1):
        assert torch.equal(back[r].double().cpu(), restored64(x[r]))


@pytest.mark.gpu
def test_container_refusals(cuda):
    codes = torch.zeros(2, 128, dtype=torch.int8, device=cuda)
    exps = torch.zeros(2, 4, dtype=torch.uint8, device=cuda)
    mhc.Checkpoint8(codes, exps, (2, 100), F32)
    for args in ((codes, exps, (3, 100), F32), (codes, exps, (2, 129), F32), (codes.float(), exps, (2, 100), F32),
                 (codes, exps.int(), (2, 100), F32), (codes.t(), exps, (2, 100), F32),
                 (codes, exps, (2, 100), torch.float16), (codes, exps, (), F32)):
        with pytest.raises(RuntimeError, match="Checkpoint8"):
            mhc.Checkpoint8(*args)
    with pytest.raises(RuntimeError, match="float32 or bfloat16"):
        mhc.checkpoint8_pack(torch.randn(2, 8, device=cuda).half())
    with pytest.raises(RuntimeError, match="last dimension"):
        mhc.checkpoint8_pack(torch.randn(2, 0, device=cuda))
    with pytest.raises(RuntimeError, match="float32 or bfloat16"):
        mhc.checkpoint8_pack(torch.randn(2, 8, device=cuda)).unpack(torch.float64)


# ---------------------------------------------------------------------------
# RMSNorm
# ---------------------------------------------------------------------------

def _norm64(x, xh, g, w, eps):
    x, g, w = x.double(), g.double(), w.double()
    C = x.size(-1)
    r = torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
    out = x / r * w
    d, dm = (g * w * xh).sum(-1, keepdim=True), (g * w * xh).abs().sum(-1, keepdim=True)
    gx = (g * w - xh * d / (C * r * r)) / r
    gw = (g * xh / r).sum(0)
    # a sum of C terms goes through at most 64 + C / 1024 additions, r then carries
    # half of that and each value a few roundings more: 2^-16 = 256 U covers them
    tol = 256 * U * ((g * w).abs() + xh.abs() * dm / (C * r * r)) / r
    tolw = (x.size(0) + 64) * U * (g * xh / r).abs().sum(0)
    return out, gx, gw, tol, tolw


@pytest.mark.gpu
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 8), (5, 31), (2, 256), (700, 264), (333, 1280), (40, 4096),
                                       (3, 4097), (2, 7168), (2, 10248), (2, 20001), (1, 32768), (2, 40000),
                                       (1, 33001)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_rmsnorm(cuda, rows, cols, dtype):
    x, g = acts(rows, cols, seed=cols, dtype=dtype), acts(rows, cols, seed=cols + 1, dtype=dtype)
    w = torch.rand(cols, generator=torch.Generator().manual_seed(2)) + 0.5
    xd, wd = x.to(cuda).requires_grad_(True), w.to(cuda).requires_grad_(True)
    out = mhc.rmsnorm_checkpoint8(xd, wd, 1e-5)
    out.backward(g.to(cuda))
    want, gx, gw, tol, tolw = _norm64(x, restored64(x), g, w, 1e-5)
    half = UB if dtype == BF16 else 0.0
    assert out.dtype == dtype and xd.grad.dtype == dtype and wd.grad.dtype == F32
    assert bool(((out.double().cpu() - want).abs() <= (64 * U + half * (1 + UB)) * want.abs()).all())
    assert bool(((xd.grad.double().cpu() - gx).abs() <= tol + half * (gx.abs() + tol)).all())
    assert bool(((wd.grad.double().cpu() - gw).abs() <= tolw).all())


@pytest.mark.gpu
def test_rmsnorm_of_many_rows_is_reproducible(cuda):
    x, g, w = acts(5000, 260, seed=1).to(cuda), acts(5000, 260, seed=2).to(cuda), torch.ones(260, device=cuda)
    a, b = (mhc.rmsnorm_checkpoint8_bwd(g, k, w, r) for _, r, k in [mhc.rmsnorm_checkpoint8_fwd(x, w)] * 2)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    out, rms, kept = mhc.rmsnorm_checkpoint8_fwd(x, w)
    assert torch.equal(kept.codes, mhc.checkpoint8_pack(x).codes)
    assert torch.equal(kept.exponents, mhc.checkpoint8_pack(x).exponents)
    _, gx, gw, tol, tolw = _norm64(x.cpu(), restored64(x), g.cpu(), w.cpu(), 1e-5)
    assert bool(((a[1].double().cpu() - gw).abs() <= tolw).all())
    assert bool(((a[0].double().cpu() - gx).abs() <= tol).all())


@pytest.mark.gpu
def test_rmsnorm_edges(cuda):
    w = torch.rand(40, device=cuda) + 0.5
    x = torch.zeros(3, 40, device=cuda)
    x[1] = 1e-30
    out, rms, kept = mhc.rmsnorm_checkpoint8_fwd(x, w)
    gx, gw = mhc.rmsnorm_checkpoint8_bwd(torch.ones_like(x), kept, w, rms)
    assert torch.isfinite(out).all() and torch.isfinite(gx).all() and torch.isfinite(gw).all()
    x[2, 5] = float("nan")
    out, rms, kept = mhc.rmsnorm_checkpoint8_fwd(x, w)
    gx, gw = mhc.rmsnorm_checkpoint8_bwd(torch.ones_like(x), kept, w, rms)
    assert torch.isnan(out[2]).all() and torch.isnan(gx[2]).all() and torch.isfinite(gx[:2]).all()
    out, rms, kept = mhc.rmsnorm_checkpoint8_fwd(x[:0], w)
    gx, gw = mhc.rmsnorm_checkpoint8_bwd(x[:0], kept, w, rms)
    assert gx.shape == (0, 40) and not gw.any()
    with pytest.raises(RuntimeError, match="Weight"):
        mhc.rmsnorm_checkpoint8(x, w[:39])
    with pytest.raises(RuntimeError, match="shape"):
        mhc.rmsnorm_checkpoint8_bwd(torch.ones(2, 40, device=cuda), mhc.checkpoint8_pack(x), w, rms)
    with pytest.raises(RuntimeError, match="float32 or bfloat16"):
        mhc.rmsnorm_checkpoint8(x.double(), w)


@pytest.mark.gpu
def test_rmsnorm_against_differences(cuda):
    """At inputs that 8 bits hold exactly, the gradient is the norm's own."""
    x = restored64(acts(6, 96, seed=8))
    g, w, v = acts(6, 96, seed=9).double(), torch.rand(96, dtype=torch.float64) + 0.5, acts(6, 96, seed=10).double()
    xd = x.float().to(cuda).requires_grad_(True)
    wd = w.float().to(cuda).requires_grad_(True)
    mhc.rmsnorm_checkpoint8(xd, wd).backward(g.float().to(cuda))

    def loss(x, w):
        return (g * x / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-5) * w).sum()

    h = 1e-5  # third derivatives of order 1: error ~ h^2 of the size of the terms, rounding 1e-16 / h
    slope = (loss(x + h * v, w.float().double()) - loss(x - h * v, w.float().double())) / (2 * h)
    got = (xd.grad.double().cpu() * v).sum()
    assert abs(slope - got) <= 256 * U * (xd.grad.double().cpu() * v).abs().sum() + 1e-6
    vw = torch.randn(96, dtype=torch.float64, generator=torch.Generator().manual_seed(1))
    slope = (loss(x, w + h * vw) - loss(x, w - h * vw)) / (2 * h)
    got = (wd.grad.double().cpu() * vw).sum()
    assert abs(slope - got) <= 256 * U * (wd.grad.double().cpu() * vw).abs().sum() + 1e-6


# ---------------------------------------------------------------------------
# weight gradient
# ---------------------------------------------------------------------------

def _wgrad_check(got, g, xh, bf16):
    g, xh = g.double().to(got.device).reshape(-1, g.size(-1)), xh.to(got.device).reshape(-1, xh.size(-1))
    T = g.size(0)
    want, mag = g.t() @ xh, g.abs().t() @ xh.abs()
    err = (got.double() - want).abs()
    # each of T additions rounds (or truncates: twice that) a partial sum of at most `mag`
    tol = 2 * (T + 8) * U * mag + (UB * (1 + UB) * want.abs() if bf16 else 0)
    assert bool((err <= tol).all()), f"max excess {(err - tol).max():.3g}"
    # over the whole matrix: T roundings of random sign, and at most one truncation in 16 terms
    bound = (T ** 0.5 + T / 16 + 8) * U * mag.norm() + (UB * want.norm() if bf16 else 0)
    assert float((got.double() - want).norm()) <= float(bound)


@pytest.mark.gpu
@pytest.mark.parametrize("T,O,K", [(1, 8, 8), (2, 1, 1), (16, 64, 128), (63, 130, 100), (64, 128, 128), (65, 129, 257),
                                   (200, 40, 1000), (1000, 300, 136), (129, 256, 512), (5, 2056, 24), (300, 1000, 33),
                                   (4100, 260, 260)])
@pytest.mark.parametrize("tg,tw", [(BF16, F32), (BF16, BF16), (F32, F32), (F32, BF16)])
def test_weight_grad(cuda, T, O, K, tg, tw):
    x, g = acts(T, K, seed=T + K), acts(T, O, seed=O, dtype=tg)
    kept = mhc.checkpoint8_pack(x.to(cuda))
    got = mhc.checkpoint8_weight_grad(g.to(cuda), kept, dtype=tw)
    assert got.shape == (O, K) and got.dtype == tw
    _wgrad_check(got, g, restored64(x), tw == BF16)
    assert torch.equal(got, mhc.checkpoint8_weight_grad(g.to(cuda), kept, dtype=tw))


@pytest.mark.gpu
@pytest.mark.parametrize("tg", [BF16, F32])
def test_weight_grad_of_many_tokens(cuda, tg):
    """A long sum of one sign, where a truncating accumulator drifts."""
    T, O, K = 33000, 136, 200
    x, g = acts(T, K, seed=1).abs(), acts(T, O, seed=2).abs().to(tg)
    got = mhc.checkpoint8_weight_grad(g.to(cuda), mhc.checkpoint8_pack(x.to(cuda)))
    xh = restored64(x).to(cuda)
    want = g.double().to(cuda).t() @ xh
    # sums of at most 4096 tokens in 16-token steps, each truncated, added in fp32
    assert float(((got.double() - want).abs() / want).max()) <= (2 * 4096 / 16 + 64) * U


@pytest.mark.gpu
@pytest.mark.parametrize("tg,tw,T,O,K", [(BF16, F32, 8192, 4096, 4096), (BF16, BF16, 16384, 4096, 2048),
                                         (F32, F32, 4096, 2048, 4096)])
def test_weight_grad_on_a_full_gpu(cuda, tg, tw, T, O, K):
    """Every SM at work, call after call: each stage's hand-overs between the
    copies, the expanding warps and the MMAs have to hold under contention."""
    x = torch.randn(T, K, device=cuda, generator=torch.Generator(device=cuda).manual_seed(1))
    g = torch.randn(T, O, device=cuda, generator=torch.Generator(device=cuda).manual_seed(2)).to(tg)
    kept = mhc.checkpoint8_pack(x)
    first = mhc.checkpoint8_weight_grad(g, kept, dtype=tw)
    _wgrad_check(first, g, kept.unpack().double(), tw == BF16)
    for _ in range(40):
        assert torch.equal(mhc.checkpoint8_weight_grad(g, kept, dtype=tw), first)


@pytest.mark.gpu
@pytest.mark.parametrize("tg", [BF16, F32])
def test_weight_grad_layouts(cuda, tg):
    x, wide = acts(150, 72, seed=1), acts(150, 400, seed=2, dtype=tg).to(cuda)
    kept = mhc.checkpoint8_pack(x.to(cuda))
    for g in (wide[:, 64:192], wide[:, 3:100], wide[:, 1:2], wide[:, :128].t().contiguous().t(),
              wide[:1].expand(150, 400), wide[:, :1].expand(150, 9)):
        _wgrad_check(mhc.checkpoint8_weight_grad(g, kept), g.cpu(), restored64(x), False)
    deep = mhc.checkpoint8_pack(x.view(5, 30, 72).to(cuda))
    _wgrad_check(mhc.checkpoint8_weight_grad(wide.view(5, 30, 400), deep), wide.cpu(), restored64(x), False)
    none = mhc.checkpoint8_pack(x[:0].to(cuda))
    assert not mhc.checkpoint8_weight_grad(wide[:0], none).any()
    with pytest.raises(RuntimeError, match="grad_out"):
        mhc.checkpoint8_weight_grad(wide[:149], kept)
    with pytest.raises(RuntimeError, match="float32 or bfloat16"):
        mhc.checkpoint8_weight_grad(wide.half(), kept)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = mhc.checkpoint8_weight_grad(wide, kept)
    side.synchronize()
    _wgrad_check(got, wide.cpu(), restored64(x), False)


@pytest.mark.gpu
@pytest.mark.parametrize("tg", [BF16, F32])
def test_weight_grad_bad_values_stay_in_their_place(cuda, tg):
    """An infinity or NaN reaches its own row of g / block of columns only."""
    x, g = acts(40, 160, seed=1), acts(40, 24, seed=2, dtype=tg)
    x[7, 70] = float("inf")  # block 2: columns 64 .. 95
    g[9, 3] = float("nan")
    got = mhc.checkpoint8_weight_grad(g.to(cuda), mhc.checkpoint8_pack(x.to(cuda))).cpu()
    bad = torch.zeros(24, 160, dtype=torch.bool)
    bad[:, 64:96] = True
    bad[3] = True
    assert torch.equal(~torch.isfinite(got), bad)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_linear(cuda, dtype):
    x, w = acts(3, 50, 96, seed=1, dtype=dtype), (acts(40, 96, seed=2) * 0.1).to(dtype)
    b, g = acts(40, seed=3, dtype=dtype), acts(3, 50, 40, seed=4, dtype=dtype)
    xs, ws, bs = (t.to(cuda).requires_grad_(True) for t in (x, w, b))
    out = mhc.linear_checkpoint8(xs, ws, bs)
    out.backward(g.to(cuda))
    assert torch.equal(out, torch.nn.functional.linear(xs, ws, bs))
    assert ws.grad.dtype == dtype and xs.grad.dtype == dtype and bs.grad.dtype == dtype
    _wgrad_check(ws.grad, g, restored64(x), dtype == BF16)
    assert torch.equal(xs.grad, g.to(cuda) @ ws)
    frozen = mhc.linear_checkpoint8(x.to(cuda), w.to(cuda).requires_grad_(True))
    frozen.sum().backward()  # an expanded gradient
    with pytest.raises(RuntimeError, match="one type"):
        mhc.linear_checkpoint8(xs, ws.double())


# ---------------------------------------------------------------------------
# recomputation
# ---------------------------------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("n,dynamic,bf16", [(4, True, False), (4, True, True), (8, True, False), (4, False, False),
                                            (12, False, False)])
def test_layer_keeps_its_streams_in_8_bits(cuda, n, dynamic, bf16):
    """The gradients are, bit for bit, those of the layer at the restored input."""
    torch.manual_seed(n)
    layer = mhc.MHCLayer(128, n, use_dynamic_h=dynamic, alpha_init=0.3, bf16_io=bf16).to(cuda)
    kept = mhc.MHCLayer(128, n, use_dynamic_h=dynamic, alpha_init=0.3, bf16_io=bf16, checkpoint_8bit=True).to(cuda)
    kept.load_state_dict(layer.state_dict())
    x = acts(40, n, 128, seed=n, dtype=BF16 if bf16 else F32).to(cuda)
    g = acts(40, n, 128, seed=5, dtype=BF16 if bf16 else F32).to(cuda)
    with torch.no_grad():
        assert torch.equal(kept(x), layer(x))
    xs = x.clone().requires_grad_(True)
    out = kept(xs)
    assert torch.equal(out, layer(x))
    out.backward(g)
    xh = mhc.checkpoint8_pack(x).unpack().requires_grad_(True)
    layer(xh).backward(g)
    assert torch.equal(xs.grad, xh.grad)
    for (name, p), q in zip(kept.named_parameters(), layer.parameters()):
        assert torch.equal(p.grad, q.grad), name


@pytest.mark.gpu
def test_layer_keeps_less(cuda):
    x = torch.randn(2048, 4, 512, device=cuda, requires_grad=True)

    def held(layer):
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        out = layer(x * 1.0)
        size = torch.cuda.memory_allocated() - before - out.numel() * 4
        del out
        return size

    full = held(mhc.MHCLayer(512, 4).to(cuda))
    kept = held(mhc.MHCLayer(512, 4, checkpoint_8bit=True).to(cuda))
    assert kept <= x.numel() * 33 / 32 + 4096 and full >= x.numel() * 4


@pytest.mark.gpu
def test_wrapper_keeps_residual_and_branch_in_8_bits(cuda):
    torch.manual_seed(3)
    plain = mhc.MHCResidualWrapper(64, 4, alpha_init=0.2).to(cuda)
    kept = mhc.MHCResidualWrapper(64, 4, alpha_init=0.2, checkpoint_8bit=True).to(cuda)
    kept.load_state_dict(plain.state_dict())
    r, b = acts(3, 20, 64, seed=1).to(cuda), acts(3, 20, 64, seed=2).to(cuda)
    w = (torch.rand(64, device=cuda) + 0.5)
    g = acts(3, 20, 64, seed=3).to(cuda)
    rs, bs = (t.clone().requires_grad_(True) for t in (r, b))
    kept(rs, bs).backward(g)
    rh, bh = (mhc.checkpoint8_pack(t).unpack().requires_grad_(True) for t in (r, b))
    plain(rh, bh).backward(g)
    assert torch.equal(rs.grad, rh.grad) and torch.equal(bs.grad, bh.grad)
    for p, q in zip(kept.parameters(), plain.parameters()):
        assert torch.equal(p.grad, q.grad)
    hidden, normed = kept.forward_prenorm(rs, bs, w)
    assert torch.equal(hidden, plain(r, b))
    assert torch.allclose(normed, mhc.rmsnorm(hidden.reshape(-1, 64), w).view_as(normed), rtol=1e-5, atol=1e-6)
    (hidden.sum() + normed.sum()).backward()


@pytest.mark.gpu
def test_recompute_of_any_function(cuda):
    x, w = acts(9, 40, seed=1).to(cuda).requires_grad_(True), acts(7, 40, seed=2).to(cuda).requires_grad_(True)
    s = torch.tensor(2.0, device=cuda)

    def f(x, w, s):
        return torch.tanh(x @ w.t()) * s, (x * x).sum(-1)

    a, b = mhc.checkpoint8_recompute(f, x, w, s)
    ra, rb = f(x, w, s)
    assert torch.equal(a, ra) and torch.equal(b, rb)
    a.sum().backward()  # the second output is not used
    xh = mhc.checkpoint8_pack(x).unpack().requires_grad_(True)
    wh = w.detach().clone().requires_grad_(True)
    f(xh, wh, s)[0].sum().backward()
    assert torch.equal(x.grad, xh.grad) and torch.equal(w.grad, wh.grad)
    with torch.no_grad():
        assert torch.equal(mhc.checkpoint8_recompute(f, x, w, s)[0], ra)


@pytest.mark.gpu
def test_autocast(cuda):
    """The linear layer casts as torch's does, and what runs again runs under the
    forward's autocast."""
    x, w = acts(30, 64, seed=1).to(cuda).requires_grad_(True), acts(24, 64, seed=2).to(cuda).requires_grad_(True)
    with torch.autocast("cuda", dtype=BF16):
        out = mhc.linear_checkpoint8(x, w)
        assert out.dtype == BF16 and torch.equal(out, torch.nn.functional.linear(x, w))
        again = mhc.checkpoint8_recompute(torch.nn.functional.linear, x, w)
    g = acts(30, 24, seed=3, dtype=BF16).to(cuda)
    out.backward(g)
    assert x.grad.dtype == F32 and w.grad.dtype == F32
    _wgrad_check(w.grad, g.cpu(), restored64(x.detach().to(BF16)), True)
    w.grad = None
    again.backward(g)  # outside of autocast
    xh = mhc.checkpoint8_pack(x).unpack()
    _wgrad_check(w.grad, g.cpu(), xh.double().cpu(), True)


@pytest.mark.gpu
def test_recompute_without_gradients_keeps_nothing(cuda):
    x = acts(9, 40, seed=1).to(cuda)
    assert mhc.checkpoint8_recompute(torch.tanh, x).grad_fn is None


@pytest.mark.gpu
@pytest.mark.parametrize("n,dynamic,bf16,training", [(4, False, True, True), (8, False, True, True),
                                                     (4, False, True, False), (4, False, False, False),
                                                     (4, True, True, False), (4, True, False, False)])
def test_layer_in_8_bits_runs_the_plain_layers_pass(cuda, n, dynamic, bf16, training):
    """With gradients on, in training and in eval mode, the result has the plain
    layer's type and bits, and so have the gradients at the restored input."""
    torch.manual_seed(n)
    layer = mhc.MHCLayer(128, n, use_dynamic_h=dynamic, alpha_init=0.3, bf16_io=bf16).to(cuda).train(training)
    kept = mhc.MHCLayer(128, n, use_dynamic_h=dynamic, alpha_init=0.3, bf16_io=bf16,
                        checkpoint_8bit=True).to(cuda).train(training)
    kept.load_state_dict(layer.state_dict())
    x = acts(40, n, 128, seed=n, dtype=BF16 if bf16 else F32).to(cuda)
    xs = x.clone().requires_grad_(True)
    out, want = kept(xs), layer(x.clone().requires_grad_(True))
    assert out.dtype == want.dtype and torch.equal(out, want)
    g = acts(40, n, 128, seed=5, dtype=want.dtype).to(cuda)
    out.backward(g)
    xh = mhc.checkpoint8_pack(x).unpack().requires_grad_(True)
    layer(xh).backward(g)
    assert torch.equal(xs.grad, xh.grad)
    for (name, p), q in zip(kept.named_parameters(), layer.named_parameters()):
        assert torch.equal(p.grad, q[1].grad), name


@pytest.mark.gpu
def test_recompute_runs_both_passes_in_one_mode(cuda):
    """The function sees gradients on in both passes, and its first pass holds nothing."""
    modes = []

    def f(t):
        modes.append(torch.is_grad_enabled())
        return torch.tanh(t) if torch.is_grad_enabled() else t.sign()

    x = acts(2048, 256, seed=1).to(cuda).requires_grad_(True)
    mhc.checkpoint8_recompute(f, x).sum().backward()
    assert modes == [True, True]
    xh = mhc.checkpoint8_pack(x).unpack().requires_grad_(True)
    torch.tanh(xh).sum().backward()
    assert torch.equal(x.grad, xh.grad)
    before = torch.cuda.memory_allocated()
    out = mhc.checkpoint8_recompute(lambda t: torch.tanh(torch.tanh(t)), x)
    assert torch.cuda.memory_allocated() - before <= out.numel() * 4 + x.numel() * 33 // 32 + 4096
    with pytest.raises(RuntimeError, match="differentiate"):
        mhc.checkpoint8_recompute(lambda t: torch.autograd.grad(torch.tanh(t).sum(), t)[0], x)


@pytest.mark.gpu
@pytest.mark.parametrize("shapes", [((2, 40000), (2, 33001), (1, 49152)), ((1184, 4096), (1184, 1032), (1184, 7168))])
def test_rmsnorm_backward_from_several_host_threads(cuda, shapes):
    """Calls of other widths in other threads, each on its own stream, take
    nothing from each other (the kernels' limits on shared memory belong to the
    process).  The entry point itself in a tight loop, so that calls overlap."""
    import threading
    lib = _C.load()

    def case(rows, cols):
        gen = torch.Generator(device=cuda).manual_seed(cols)
        x, g = (torch.randn(rows, cols, device=cuda, generator=gen, dtype=BF16) for _ in range(2))
        w = torch.rand(cols, device=cuda, generator=gen) + 0.5
        _, rms, kept = mhc.rmsnorm_checkpoint8_fwd(x, w)
        want = mhc.rmsnorm_checkpoint8_bwd(g, kept, w, rms)
        got = torch.empty_like(want[0]), torch.empty_like(want[1])
        size = lib.mhc_rmsnorm_checkpoint8_bwd_workspace_bytes(rows, cols)
        ws, stream = torch.empty(size, dtype=torch.uint8, device=cuda), torch.cuda.Stream()
        held = (g, kept, w, rms, ws, stream)
        args = (g.data_ptr(), 1, kept.codes.data_ptr(), kept.exponents.data_ptr(), w.data_ptr(), rms.data_ptr(),
                got[0].data_ptr(), got[1].data_ptr(), rows, cols, ws.data_ptr(), size, stream.cuda_stream)
        return args, got, want, held

    cases = [case(*s) for s in shapes]
    torch.cuda.synchronize()
    errors = []

    def work(args):
        for _ in range(2000):
            if lib.mhc_rmsnorm_checkpoint8_bwd(*args):
                errors.append(_C.last_error())
                return

    threads = [threading.Thread(target=work, args=(c[0],)) for c in cases]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not errors, errors
    for _, got, want, _ in cases:
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.gpu
def test_second_derivatives_raise(cuda):
    """The kernels' gradients have no graph: differentiating one again raises
    instead of leaving terms out."""
    x, w = acts(9, 32, seed=1).to(cuda).requires_grad_(True), acts(7, 32, seed=2).to(cuda).requires_grad_(True)
    v, ids = torch.ones(32, device=cuda, requires_grad=True), torch.arange(7, device=cuda)
    for out, by in ((mhc.linear_checkpoint8(x, w), x), (mhc.linear_checkpoint8(x, w), w),
                    (mhc.rmsnorm_checkpoint8(x, v), x), (mhc.checkpoint8_recompute(torch.tanh, x), x),
                    (mhc.stream_embedding(ids, w, 2), w)):
        grad, = torch.autograd.grad(out.square().sum(), by, create_graph=True)
        with pytest.raises(RuntimeError, match="once_differentiable"):
            grad.sum().backward()


@pytest.mark.gpu
def test_recompute_refuses_results_that_have_no_gradient(cuda):
    """A list or a dict would pass through autograd without a graph."""
    x = acts(9, 40, seed=1).to(cuda).requires_grad_(True)
    for pack in (lambda t: [t * 2], lambda t: {"out": t * 2}, lambda t: (t * 2, [t])):
        with pytest.raises(RuntimeError, match="tuple of tensors"):
            mhc.checkpoint8_recompute(pack, x)
    out, none, five, names = mhc.checkpoint8_recompute(lambda t: (t * 2, None, 5, ["a"]), x)
    assert none is None and five == 5 and names == ["a"]
    out.sum().backward()
    assert torch.equal(x.grad, torch.full_like(x, 2.0))


@pytest.mark.gpu
@pytest.mark.parametrize("mode", ["frozen", "no_grad", "autocast"])
def test_linear_keeps_nothing_for_a_frozen_weight(cuda, mode):
    """Without a weight gradient to come, x is neither packed nor kept."""
    x, w = acts(4096, 512, seed=1).to(cuda).requires_grad_(True), (acts(64, 512, seed=2) * 0.1).to(cuda)
    b = acts(64, seed=3).to(cuda).requires_grad_(True)
    if mode == "no_grad":
        w.requires_grad_(True)
    with torch.set_grad_enabled(mode != "no_grad"), torch.autocast("cuda", dtype=BF16, enabled=mode == "autocast"):
        mhc.linear_checkpoint8(x, w, b)  # the library's own buffers
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats()
        before = torch.cuda.memory_allocated()
        out = mhc.linear_checkpoint8(x, w, b)
        held, peak = torch.cuda.memory_allocated() - before, torch.cuda.max_memory_allocated() - before
        assert torch.equal(out, torch.nn.functional.linear(x, w, b))
    assert held <= out.numel() * 4 + w.numel() * 4 + 8192  # autocast keeps w's copy
    if mode != "autocast":
        assert peak <= 2 * out.numel() * 4 + 8192
    if mode == "no_grad":
        assert out.grad_fn is None
        return
    g = acts(4096, 64, seed=4, dtype=out.dtype).to(cuda)
    out.backward(g)
    xs, bs = (t.detach().clone().requires_grad_(True) for t in (x, b))
    with torch.autocast("cuda", dtype=BF16, enabled=mode == "autocast"):
        torch.nn.functional.linear(xs, w, bs).backward(g)
    assert torch.equal(x.grad, xs.grad) and torch.equal(b.grad, bs.grad)


@pytest.mark.gpu
def test_linear_refuses_a_weight_vector(cuda):
    """Before the forward pass, not in the backward."""
    x, w = torch.randn(8, 8, device=cuda), torch.randn(8, device=cuda, requires_grad=True)
    with pytest.raises(RuntimeError, match="weight must be"):
        mhc.linear_checkpoint8(x, w)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [4, 3])
def test_wrapper_in_8_bits_without_gradients_is_the_plain_one(cuda, n):
    """Output and norm in one pass where the plain wrapper has it, and no packing."""
    torch.manual_seed(3)
    plain = mhc.MHCResidualWrapper(64, n, alpha_init=0.2).to(cuda).eval()
    kept = mhc.MHCResidualWrapper(64, n, alpha_init=0.2, checkpoint_8bit=True).to(cuda).eval()
    kept.load_state_dict(plain.state_dict())
    r, b, w = acts(3, 20, 64, seed=1).to(cuda), acts(3, 20, 64, seed=2).to(cuda), torch.rand(64, device=cuda) + 0.5

    def launches(wrapper):
        with torch.no_grad():
            _C.profile_enable(True)
            try:
                out = wrapper.forward_prenorm(r, b, w)
                torch.cuda.synchronize()
                return out, sorted(_C.profile_report())
            finally:
                _C.profile_enable(False)

    (hidden, normed), names = launches(kept)
    (want, want_normed), want_names = launches(plain)
    assert torch.equal(hidden, want) and torch.equal(normed, want_normed)
    assert names == want_names and not any("checkpoint8" in k for k in names)


def test_modules_pickled_before_the_flag_still_run():
    layer = mhc.MHCLayer(64, 4)
    state = dict(layer.__dict__)
    del state["checkpoint_8bit"]
    old = mhc.MHCLayer.__new__(mhc.MHCLayer)
    old.__setstate__(state)  # as unpickling does
    assert old.checkpoint_8bit is False
    with pytest.raises(RuntimeError, match="CUDA"):
        old(torch.randn(2, 4, 64))


@pytest.mark.gpu
@pytest.mark.parametrize("per_sm,more,cols", [(8, 0, 1032), (8, -1, 1032), (8, -1, 4096), (8, 0, 4096), (16, 132, 1280),
                                              (33, 116, 2048), (20, 41, 4096), (16, 32, 7168), (8, 117, 8192),
                                              (8, 1, 8200), (9, 0, 1928)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_rmsnorm_backward_of_training_batches(cuda, per_sm, more, cols, dtype):
    """Rows enough that a block meets several of them: from 8 rows an SM and 1025
    to 8192 columns on over a ring of rows in shared memory, whose places are
    filled again and again; one row less and a wider row take other kernels."""
    rows = per_sm * torch.cuda.get_device_properties(cuda).multi_processor_count + more
    gen = torch.Generator(device=cuda).manual_seed(rows + cols)
    loud = torch.exp(torch.randn(cols, device=cuda, generator=gen))
    x, g = ((torch.randn(rows, cols, device=cuda, generator=gen) * loud).to(dtype) for _ in range(2))
    w = torch.rand(cols, device=cuda, generator=gen) + 0.5
    _, rms, kept = mhc.rmsnorm_checkpoint8_fwd(x, w)
    gx, gw = mhc.rmsnorm_checkpoint8_bwd(g, kept, w, rms)
    _, want, want_w, tol, tolw = _norm64(x, kept.unpack().double(), g, w, 1e-5)
    half = UB if dtype == BF16 else 0.0
    assert bool(((gx.double() - want).abs() <= tol + half * (want.abs() + tol)).all())
    assert bool(((gw.double() - want_w).abs() <= tolw).all())
    for _ in range(3):
        again = mhc.rmsnorm_checkpoint8_bwd(g, kept, w, rms)
        assert torch.equal(again[0], gx) and torch.equal(again[1], gw)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,cols", [(700, 33001), (700, 40000), (601, 49152), (601, 49160), (333, 50001)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_rmsnorm_backward_of_many_long_rows(cuda, rows, cols, dtype):
    """Rows past the registers, several a block; past 49152 columns the weight's
    share is kept outside of shared memory."""
    gen = torch.Generator(device=cuda).manual_seed(cols)
    x, g = (torch.randn(rows, cols, device=cuda, generator=gen).to(dtype) for _ in range(2))
    w = torch.rand(cols, device=cuda, generator=gen) + 0.5
    _, rms, kept = mhc.rmsnorm_checkpoint8_fwd(x, w)
    gx, gw = mhc.rmsnorm_checkpoint8_bwd(g, kept, w, rms)
    _, want, want_w, tol, tolw = _norm64(x, kept.unpack().double(), g, w, 1e-5)
    half = UB if dtype == BF16 else 0.0
    assert bool(((gx.double() - want).abs() <= tol + half * (want.abs() + tol)).all())
    assert bool(((gw.double() - want_w).abs() <= tolw).all())
    again = mhc.rmsnorm_checkpoint8_bwd(g, kept, w, rms)
    assert torch.equal(again[0], gx) and torch.equal(again[1], gw)
