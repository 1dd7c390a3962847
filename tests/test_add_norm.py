"""Residual addition with RMSNorm, its gradients and its 8-bit outputs, against the
formulas in 64 bits."""
import ctypes

import pytest
import torch

import mhc_ascend_b200 as mhc
from mhc_ascend_b200 import _C

U = 2.0 ** -24  # unit roundoff of fp32
UB = 2.0 ** -8  # of bf16: 8 significant bits against 24
F32, BF16 = torch.float32, torch.bfloat16
E4M3, INT8 = torch.float8_e4m3fn, torch.int8
EPS = 1e-5


def half_step(t, dtype):
    """Rounding to `dtype`, relative to the value."""
    return (UB if dtype == BF16 else U) * t.abs()


def terms(C):
    """Additions behind a row's sum: a thread's own values (32 at most in registers,
    every 4096th unit's in the long kernels), then two levels of five in the tree."""
    return max(32, C // 512) + 12


def inputs(R, C, tr, tb, seed=0):
    gen = torch.Generator().manual_seed(1000 * R + C + seed)
    rand = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    return (rand(R, C) * 2).to(tr), rand(R, C).to(tb), 0.5 + torch.rand(C, generator=gen), rand(R, C).to(tr), rand(R, C).to(tb)


def norm64(h, w, eps=EPS):
    h = h.double()
    r = (h.pow(2).mean(1, keepdim=True) + eps).sqrt()
    return h / r * w.double(), r


SIZES = [(1, 1), (3, 7), (5, 8), (2, 9), (17, 100), (9, 128), (4, 129), (33, 256), (8, 264), (7, 512), (5, 1000), (3, 1024),
         (4, 1025), (6, 1032), (5, 2048), (3, 2056), (2, 4096), (600, 1100), (700, 264), (3, 4097), (2, 7168), (2, 8192), (3, 8200),
         (2, 8191), (300, 2048), (310, 4104), (300, 8192), (2, 32768), (2, 32776), (5, 251), (67, 500), (9, 1015), (7, 1017), (5, 1019), (3, 9001), (4, 20002), (3, 32759), (3, 32761), (3, 50001), (2, 49160)]


# ---------------------------------------------------------------------------
# no GPU needed
# ---------------------------------------------------------------------------

def test_cpu_tensors_raise():
    x, w = torch.randn(2, 8), torch.ones(8)
    for call in (lambda: mhc.add_rmsnorm(x, x, w), lambda: mhc.add_rmsnorm_quantized(x, x, w),
                 lambda: mhc.add_rmsnorm_bwd(None, x, x, w, torch.ones(2)), lambda: mhc.Coded8(x.to(E4M3), torch.ones(2))):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()


def test_entry_points_validate_without_gpu():
    lib = _C.load()
    p, odd = ctypes.c_void_p(16), ctypes.c_void_p(20)

    def fwd(res=p, br=p, w=p, h=p, out=p, codes=None, exps=None, R=4, C=8, eps=1e-5, drop=0, state=None):
        return lib.mhc_add_rmsnorm_fwd(res, 0, br, 0, w, h, out, None, codes, exps, R, C, eps, drop, state, 0, 0, None)

    assert fwd(R=0) == 0
    assert fwd(R=-1) == -1 and fwd(C=0) == -1 and fwd(eps=-1.0) == -1 and "eps" in _C.last_error()
    assert fwd(res=None) == -1 and fwd(br=None) == -1 and fwd(w=None) == -1 and fwd(h=None) == -1 and fwd(out=None) == -1
    assert fwd(R=1 << 31) == -2 and fwd(C=(1 << 30) + 1) == -2
    assert fwd(drop=-1) == -1 and fwd(drop=65537) == -1 and fwd(state=odd) == -3
    assert fwd(codes=p) == -1 and "together" in _C.last_error()
    assert fwd(codes=odd, exps=p) == -3

    def coded(codes=p, scales=p, R=4, C=8):
        return lib.mhc_add_rmsnorm_coded(p, 0, p, 1, p, p, codes, 0, scales, 1, R, C, 1e-5, None)

    assert coded(R=0) == 0 and coded(codes=None) == -1 and coded(scales=None) == -1 and coded(C=-1) == -1
    assert lib.mhc_coded8_unpack(p, 0, None, 0, p, 0, 4, 8, None) == -1
    assert lib.mhc_coded8_unpack(p, 0, p, 0, p, 0, 4, 0, None) == -1

    def bwd(gh=p, g=p, h=p, gr=p, gw=p, rms=p, R=4, C=8, drop=0, ws=p, size=1 << 30):
        return lib.mhc_add_rmsnorm_bwd(gh, g, h, 0, 1, p, rms, gr, None, gw, R, C, drop, None, 0, 0, ws, size, None)

    assert bwd(g=None) == -1 and bwd(h=None) == -1 and bwd(gr=None) == -1 and bwd(gw=None) == -1 and bwd(rms=None) == -1
    assert bwd(R=-1) == -1 and bwd(C=0) == -1 and bwd(drop=70000) == -1
    assert bwd(ws=None) == -4 and bwd(size=16) == -4 and "workspace" in _C.last_error()
    assert lib.mhc_add_rmsnorm_bwd_workspace_bytes(-1, 8) == 0
    assert lib.mhc_add_rmsnorm_bwd_workspace_bytes(5, 4096) >= 5 * 4096 * 4


# ---------------------------------------------------------------------------
# GPU: forward
# ---------------------------------------------------------------------------

def check_out(out, hidden, w, C, dtype):
    want, _ = norm64(hidden, w)
    # the sum's additions at half weight (root), then mean, eps, root, reciprocal, two products and their inputs
    tol = (0.5 * terms(C) + 7) * U * want.abs() + half_step(want, dtype) * (1 + 64 * U)
    err = (out.double() - want).abs()
    assert bool((err <= tol).all()), f"max excess {(err - tol).max():.3g}"


@pytest.mark.gpu
@pytest.mark.parametrize("tr,tb", [(F32, F32), (F32, BF16), (BF16, F32), (BF16, BF16)])
@pytest.mark.parametrize("R,C", SIZES)
def test_forward(cuda, R, C, tr, tb):
    res, br, w, _, _ = inputs(R, C, tr, tb)
    hidden, out, rms, kept = mhc.add_rmsnorm_fwd(res.to(cuda), br.to(cuda), w.to(cuda), keep=True)
    assert hidden.dtype == tr and out.dtype == tb
    assert torch.equal(hidden.cpu(), (res.float() + br.float()).to(tr))  # one fp32 sum, rounded once
    check_out(out.cpu(), hidden.cpu(), w, C, tb)
    r64 = norm64(hidden.cpu(), w)[1].squeeze(1)
    assert bool(((rms.cpu().double() - r64).abs() <= (0.5 * terms(C) + 4) * U * r64).all())
    packed = mhc.checkpoint8_pack(out)
    assert torch.equal(kept.codes, packed.codes) and torch.equal(kept.exponents, packed.exponents)
    plain = mhc.add_rmsnorm_fwd(res.to(cuda), br.to(cuda), w.to(cuda))
    assert torch.equal(plain[0], hidden) and torch.equal(plain[1], out) and plain[3] is None


@pytest.mark.gpu
@pytest.mark.parametrize("tr", [F32, BF16])
@pytest.mark.parametrize("R,C", [(3, 7), (5, 1000), (4, 1025), (4, 2048), (2, 8192), (3, 8200), (2, 8201), (2, 33000)])
def test_dropout_is_the_operator_s(cuda, R, C, tr):
    """The fused mask is dropout's: with a 32-bit branch the sum is the same to the bit."""
    res, br, w, gh, go = (t.to(cuda) for t in inputs(R, C, tr, F32))
    rng = (R, 2 ** 32 - C // 16)
    hidden, out, rms, _ = mhc.add_rmsnorm_fwd(res, br, w, EPS, 0.3, rng)
    apart = mhc.add_rmsnorm_fwd(res, mhc.dropout_fwd(br, 0.3, rng), w, EPS)
    assert torch.equal(hidden, apart[0]) and torch.equal(out, apart[1])
    gr, gb, gw = mhc.add_rmsnorm_bwd(gh, go, hidden, w, rms, 0.3, rng)
    plain = mhc.add_rmsnorm_bwd(gh, go, hidden, w, rms)
    assert torch.equal(gr, plain[0]) and torch.equal(gw, plain[2])
    if tr == F32:
        assert torch.equal(gb, mhc.dropout_fwd(gr, 0.3, rng))
    state = torch.tensor(rng, device=cuda)
    again = mhc.add_rmsnorm_fwd(res, br, w, EPS, 0.3, state)
    assert torch.equal(again[0], hidden)
    assert torch.equal(mhc.add_rmsnorm_bwd(gh, go, hidden, w, rms, 0.3, state)[1], gb)
    nothing = mhc.add_rmsnorm_fwd(res, br, w, EPS, 1.0, rng)
    assert torch.equal(nothing[0], res)


@pytest.mark.gpu
def test_layouts_and_shapes(cuda):
    res, br, w, _, _ = inputs(24, 136, F32, BF16)
    want = mhc.add_rmsnorm(res.to(cuda), br.to(cuda), w.to(cuda))
    wide_r, wide_b = torch.zeros(24, 300, device=cuda), torch.zeros(136, 24, device=cuda, dtype=BF16)
    wide_r[:, 5:141], wide_b[:] = res.to(cuda), br.to(cuda).t()
    flat = torch.zeros(24 * 136 + 3, device=cuda)  # rows that start off alignment
    flat[3:] = res.to(cuda).flatten()
    for r, b in ((wide_r[:, 5:141], wide_b.t()), (flat[3:].view(24, 136), br.to(cuda))):
        for got, exp in zip(mhc.add_rmsnorm(r, b, w.to(cuda)), want):
            assert torch.equal(got, exp)
    hidden, out = mhc.add_rmsnorm(res.to(cuda).view(2, 3, 4, 136), br.to(cuda).view(2, 3, 4, 136), w.to(cuda).double())
    assert hidden.shape == (2, 3, 4, 136) and torch.equal(out.view(24, 136), want[1])
    one = mhc.add_rmsnorm(res[0].to(cuda), br[0].to(cuda), w.to(cuda))
    assert one[0].shape == (136,) and torch.equal(one[1], want[1][0])
    none = mhc.add_rmsnorm_fwd(res[:0].to(cuda), br[:0].to(cuda), w.to(cuda), keep=True)
    assert none[0].shape == (0, 136) and none[3].rows == 0


@pytest.mark.gpu
def test_rows_of_zeros_infinities_and_nans(cuda):
    x = torch.zeros(6, 300, device=cuda)
    x[1, 4], x[2, 5], x[3] = float("inf"), float("nan"), 1e30
    x[4, :] = 1e-30
    z, w = torch.zeros_like(x), torch.ones(300, device=cuda)
    _, out, _, kept = mhc.add_rmsnorm_fwd(x, z, w, keep=True)
    assert not out[0].any() and torch.isnan(out[2]).all()
    assert torch.isnan(out[1, 4]) and out[1, 5] == 0
    assert torch.equal(kept.codes, mhc.checkpoint8_pack(out).codes)
    want = x[4].double() / 1e-5 ** 0.5
    assert bool(((out[4].double() - want).abs() <= 16 * U * want).all())
    with torch.no_grad():
        for codes in (E4M3, INT8):
            for group in (None, 128):
                _, q = mhc.add_rmsnorm_quantized(x, z, w, codes=codes, group=group)
                back = q.unpack(F32)
                assert not back[0].any() and torch.isnan(back[2]).all()
                assert torch.isnan(back[1, :128]).all() and not (group and back[1, 128:].any())
                assert q.scales[0].max() == 2.0 ** -100


@pytest.mark.gpu
@pytest.mark.parametrize("codes", [E4M3, INT8])
@pytest.mark.parametrize("group", [None, 128])
@pytest.mark.parametrize("R,C,tr,tb", [(1, 1, F32, F32), (3, 9, BF16, F32), (17, 100, F32, BF16), (9, 128, BF16, BF16),
                                       (600, 264, F32, F32), (4, 1000, BF16, BF16), (4, 1025, F32, BF16), (3, 2048, BF16, BF16),
                                       (5, 4096, BF16, BF16), (2, 4097, F32, F32), (2, 7168, BF16, BF16),
                                       (2, 8200, F32, F32), (300, 1032, BF16, BF16), (301, 4000, F32, BF16),
                                       (300, 7168, BF16, BF16), (300, 8192, BF16, F32), (2, 32770, BF16, F32), (70, 251, BF16, BF16), (9, 1015, F32, BF16), (305, 2001, BF16, F32),
                                       (4, 7999, BF16, BF16), (3, 20001, F32, F32), (2, 33024, F32, BF16)])
def test_quantized(cuda, R, C, tr, tb, group, codes):
    res, br, w, _, _ = inputs(R, C, tr, tb)
    br[:, C // 2] *= 40  # a loud channel
    hidden, q = mhc.add_rmsnorm_quantized(res.to(cuda), br.to(cuda), w.to(cuda), EPS, codes, group)
    assert torch.equal(hidden.cpu(), (res.float() + br.float()).to(tr))
    y, _ = norm64(hidden.cpu(), w)
    rel = (0.5 * terms(C) + 12) * U  # the output's, and the scale's and the quotient's roundings
    G = -(-C // 128) if group else 1
    width = 128 if group else C
    padded = torch.nn.functional.pad(y, (0, G * width - C)).view(R, G, width)
    most = 448.0 if codes == E4M3 else 127.0
    scale = (padded.abs().amax(-1) / most).clamp(min=2.0 ** -100)
    assert q.codes.dtype == codes and q.scales.shape == (R, G)
    got = q.scales.cpu().double().view(R, G)
    assert bool(((got - scale).abs() <= rel * scale).all())
    step = got.repeat_interleave(width, 1)[:, :C]
    v = q.codes.cpu().float().double()
    assert v.abs().max() <= most
    # to nearest: half a step of int8; half of 2^-3 of the value, or of 2^-9, of e4m3
    half = torch.full_like(y, 0.5) if codes == INT8 else torch.maximum(v.abs(), (y / step).abs()) * 2.0 ** -4 + 2.0 ** -10
    err = (y / step - v).abs()
    tol = half + rel * (y / step).abs()
    assert bool((err <= tol).all()), f"max excess {(err - tol).max():.3g}"
    for dtype in (F32, BF16):
        exact = (q.codes.float().cpu() * q.scales.cpu().view(R, G).repeat_interleave(width, 1)[:, :C]).to(dtype)
        assert torch.equal(q.unpack(dtype).cpu(), exact)  # one fp32 product, rounded once


@pytest.mark.gpu
def test_all_codes_unpack(cuda):
    """Every e4m3 and int8 code, also in rows that wide accesses do not fit."""
    for dtype in (E4M3, INT8):
        every = torch.arange(256, dtype=torch.uint8, device=cuda).view(dtype)
        for codes in (every.view(1, 256), every[:255].view(1, 255), every[1:].view(1, 255), every[1:254].view(1, 253)):
            got = mhc.Coded8(codes, torch.full((1, 1), 0.5, device=cuda)).unpack(F32)
            assert torch.equal(torch.nan_to_num(got, 7e7), torch.nan_to_num(codes.float() * 0.5, 7e7))


# ---------------------------------------------------------------------------
# GPU: backward
# ---------------------------------------------------------------------------

def check_grads(got, gh, go, hidden, w, keep, scale, C, R):
    gr, gb, gw = (t.cpu() for t in got)
    h, g, w64 = hidden.double(), go.double(), w.double()
    r = (h.pow(2).mean(1, keepdim=True) + EPS).sqrt()
    gwt = g * w64
    d = (gwt * h).sum(1, keepdim=True)
    gi = gwt / r - h * d / (C * r ** 3)
    mag = gwt.abs() / r + h.abs() * (gwt * h).abs().sum(1, keepdim=True) / (C * r ** 3)
    if gh is not None:
        gi, mag = gi + gh.double(), mag + gh.double().abs()
    # d's additions; r (half of its sum's, cubed) and a dozen operations of each term
    tol = (terms(C) + 1.5 * terms(C) + 16) * U * mag
    err = (gr.double() - gi).abs()
    assert bool((err <= tol + half_step(gi, gr.dtype)).all()), f"residual: max excess {(err - tol).max():.3g}"
    want = gi * keep * scale
    err = (gb.double() - want).abs()
    tol = (tol + 2 * U * gi.abs()) * scale
    assert bool((err <= tol + half_step(want, gb.dtype) * (1 + 64 * U)).all()), f"branch: max excess {(err - tol).max():.3g}"
    want, mag = (g * h / r).sum(0), (g * h / r).abs().sum(0)
    tol = (R + 0.5 * terms(C) + 16) * U * mag  # R additions in some order
    err = (gw.double() - want).abs()
    assert bool((err <= tol).all()), f"weight: max excess {(err - tol).max():.3g}"


@pytest.mark.gpu
@pytest.mark.parametrize("tr,tb", [(F32, F32), (F32, BF16), (BF16, F32), (BF16, BF16)])
@pytest.mark.parametrize("R,C", SIZES + [(3000, 2048), (1300, 1025), (1200, 2050), (700, 2052), (330, 6001), (5000, 40), (5100, 41),
                                     (5003, 250), (5001, 500), (4999, 1010), (4990, 1018), (320, 12001), (310, 8194)])
def test_backward(cuda, R, C, tr, tb):
    res, br, w, gh, go = inputs(R, C, tr, tb)
    hidden, _, rms, _ = mhc.add_rmsnorm_fwd(res.to(cuda), br.to(cuda), w.to(cuda))
    p, rng = 0.3, (4, 4)
    keep = mhc.dropout_fwd(torch.ones(R, C, device=cuda), p, rng).cpu() != 0
    scale = 1 / (1 - round(p * 65536) / 65536)
    for grad in (gh, None):
        args = (None if grad is None else grad.to(cuda), go.to(cuda), hidden, w.to(cuda), rms)
        got = mhc.add_rmsnorm_bwd(*args)
        assert got[0].dtype == tr and got[1].dtype == tb and got[2].dtype == F32
        check_grads(got, grad, go, hidden.cpu(), w, 1.0, 1.0, C, R)
        assert all(torch.equal(a, b) for a, b in zip(got, mhc.add_rmsnorm_bwd(*args)))  # bitwise
    check_grads(mhc.add_rmsnorm_bwd(*args, p, rng), None, go, hidden.cpu(), w, keep, scale, C, R)


@pytest.mark.gpu
def test_backward_layouts(cuda):
    for R, C in ((40, 256), (30, 2048), (12, 8200)):
        res, br, w, gh, go = (t.to(cuda) for t in inputs(R, C, F32, BF16))
        hidden, _, rms, _ = mhc.add_rmsnorm_fwd(res, br, w)
        want = mhc.add_rmsnorm_bwd(gh, go, hidden, w, rms)
        wide = torch.zeros(R, C + 9, device=cuda)
        wide[:, 4:4 + C] = gh
        off = torch.zeros(R * C + 1, device=cuda, dtype=BF16)  # off alignment: another kernel
        off[1:] = go.flatten()
        got = mhc.add_rmsnorm_bwd(wide[:, 4:4 + C], off[1:].view(R, C), hidden, w, rms)
        check_grads(got, gh.cpu(), go.cpu(), hidden.cpu(), w.cpu(), 1.0, 1.0, C, R)
        strided = mhc.add_rmsnorm_bwd(wide[:, 4:4 + C], go.t().contiguous().t(), hidden, w, rms)
        assert all(torch.equal(a, b) for a, b in zip(strided, want))
    empty = mhc.add_rmsnorm_bwd(None, go[:0], hidden[:0], w, rms[:0])
    assert empty[0].shape == (0, C) and not empty[2].any()


@pytest.mark.gpu
@pytest.mark.parametrize("tr,tb", [(F32, BF16), (BF16, F32)])
@pytest.mark.parametrize("R,C", [(20, 100), (17, 500), (9, 1000), (5, 1500), (4, 6000), (3, 8190), (3, 20000), (2, 33000)])
def test_starts_off_alignment(cuda, R, C, tr, tb):
    """Views that begin one element into their storage: the kernels for any row."""
    def off(t):
        flat = torch.empty(t.numel() + 1, dtype=t.dtype, device=cuda)
        flat[1:] = t.flatten().to(cuda)
        return flat[1:].view(t.shape)

    res, br, w, gh, go = inputs(R, C, tr, tb)
    p, rng = 0.3, (6, 2 ** 32 - 5)
    keep = mhc.dropout_fwd(torch.ones(R, C, device=cuda), p, rng).cpu() != 0
    scale = 1 / (1 - round(p * 65536) / 65536)
    hidden, out, rms, kept = mhc.add_rmsnorm_fwd(off(res), off(br), off(w), EPS, p, rng, keep=True)
    dropped = torch.where(keep, br.float() * torch.tensor(scale).float(), 0.0)
    assert torch.equal(hidden.cpu(), (res.float() + dropped).to(tr))
    check_out(out.cpu(), hidden.cpu(), w, C, tb)
    packed = mhc.checkpoint8_pack(out)
    assert torch.equal(kept.codes, packed.codes) and torch.equal(kept.exponents, packed.exponents)
    got = mhc.add_rmsnorm_bwd(off(gh), off(go), off(hidden), off(w), rms, p, rng)
    check_grads(got, gh, go, hidden.cpu(), w, keep, scale, C, R)
    for codes in (E4M3, INT8):
        for group in (None, 128):
            h, q = mhc.add_rmsnorm_quantized(off(res), off(br), off(w), EPS, codes, group)
            want = mhc.add_rmsnorm_quantized(res.to(cuda), br.to(cuda), w.to(cuda), EPS, codes, group)
            assert torch.equal(h, want[0])
            # the same sum in another order: scales a few units apart, codes where they round the other way
            assert bool(((q.scales - want[1].scales).abs() <= 2 * (terms(C) + 12) * U * want[1].scales).all())
            step = q.scales.repeat_interleave(128 if group else C, 1)[:, :C]
            apart = (q.unpack(F32) - want[1].unpack(F32)).abs()
            assert bool((apart <= torch.clamp(q.unpack(F32).abs() * 2.0 ** -3, min=0) * 1.01 + step * 1.01).all())


@pytest.mark.gpu
def test_autograd_against_differences(cuda):
    R, C, p, rng = 6, 40, 0.25, (8, 1)
    res, br, w, gh, go = inputs(R, C, F32, F32)
    leaves = [t.to(cuda).requires_grad_(True) for t in (res, br, w)]
    hidden, out = mhc.add_rmsnorm(*leaves, EPS, p, rng)
    ((hidden * gh.to(cuda)).sum() + (out * go.to(cuda)).sum()).backward()
    mask = mhc.dropout_fwd(torch.ones(R, C, device=cuda), p, rng).cpu().double()

    def loss(r, b, v):
        h = r + b * mask
        return ((h * gh.double()).sum() + (norm64(h, v)[0] * go.double()).sum()).item()

    gen = torch.Generator().manual_seed(5)
    at = [t.double() for t in (res, br, w)]
    for i, leaf in enumerate(leaves):
        d = torch.randn(at[i].shape, generator=gen, dtype=torch.float64)
        step = 1e-5
        up, down = ([t + s * step * d if j == i else t for j, t in enumerate(at)] for s in (1, -1))
        slope = (loss(*up) - loss(*down)) / (2 * step)
        got = (leaf.grad.cpu().double() * d).sum().item()
        # third derivatives ~ 10 of 240 terms x step^2, and fp32 gradients of size ~2 with ~100 roundings
        assert got == pytest.approx(slope, abs=240 * (10 * step ** 2 + 2 * 100 * U) + 1e-6)


@pytest.mark.gpu
def test_autograd_of_one_result(cuda):
    res, br, w, gh, go = (t.to(cuda) for t in inputs(7, 520, F32, BF16))
    for use in ("hidden", "out", "both"):
        leaves = [res.clone().requires_grad_(True), br.clone().requires_grad_(True), w.clone().requires_grad_(True)]
        hidden, out = mhc.add_rmsnorm(*leaves)
        loss = 0
        if use != "out":
            loss = loss + (hidden * gh).sum()
        if use != "hidden":
            loss = loss + (out.float() * go.float()).sum()
        loss.backward()
        h, _, rms, _ = mhc.add_rmsnorm_fwd(res, br, w)
        want = mhc.add_rmsnorm_bwd(gh if use != "out" else None, go if use != "hidden" else torch.zeros_like(go), h, w, rms)
        assert all(torch.equal(t.grad, g) for t, g in zip(leaves, want))
        assert use != "hidden" or torch.equal(leaves[0].grad, gh)
    same = res.clone().requires_grad_(True)  # one tensor as both inputs
    hidden, out = mhc.add_rmsnorm(same, same, w)
    out.backward(go.float())
    h, _, rms, _ = mhc.add_rmsnorm_fwd(res, res, w)
    gr, gb, _ = mhc.add_rmsnorm_bwd(None, go.float(), h, w, rms)
    assert torch.equal(same.grad, gr + gb)


@pytest.mark.gpu
def test_kept_output_feeds_the_linear_layer(cuda):
    """The 8-bit output in place of the linear layer's own packing: the same gradients."""
    res, br, w, _, _ = (t.to(cuda) for t in inputs(96, 256, F32, F32))
    W = torch.randn(64, 256, device=cuda)
    grads = []
    for keep in (True, False):
        leaves = [t.clone().requires_grad_(True) for t in (res, br, w, W)]
        if keep:
            hidden, out, kept = mhc.add_rmsnorm(*leaves[:3], keep=True)
            y = mhc.linear_checkpoint8(out, leaves[3], kept=kept)
        else:
            hidden, out = mhc.add_rmsnorm(*leaves[:3])
            y = mhc.linear_checkpoint8(out, leaves[3])
        (y.square().sum() + hidden.sum()).backward()
        grads.append([t.grad for t in leaves])
    assert all(torch.equal(a, b) for a, b in zip(*grads))
    with pytest.raises(RuntimeError, match="kept must be"):
        mhc.linear_checkpoint8(out[:5], leaves[3], kept=kept)


@pytest.mark.gpu
def test_captured_step_on_another_stream(cuda):
    res, br, w, gh, go = (t.to(cuda) for t in inputs(300, 2048, F32, BF16))
    counter = mhc.DropoutCounter(3).to(cuda)
    groups = mhc.dropout_groups(br.shape)

    def step():
        rng = counter.take(groups)
        hidden, out, rms, kept = mhc.add_rmsnorm_fwd(res, br, w, EPS, 0.2, rng, keep=True)
        return hidden, out, kept.codes, *mhc.add_rmsnorm_bwd(gh, go, hidden, w, rms, 0.2, rng)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for turn in (1, 2):
        graph.replay()
        counter.state[1] = groups * turn
        want = step()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.gpu
def test_widths_from_several_host_threads(cuda):
    """Calls of several widths at once, each thread on a stream of its own: a kernel's limit
    on shared memory belongs to the process, and so may not follow one call's width."""
    import threading
    work, errors = [], []
    for R, C, tr, tb in ((40, 1032, F32, BF16), (40, 8192, F32, F32), (6, 28672, BF16, BF16), (6, 20001, F32, BF16)):
        res, br, w, gh, go = (t.to(cuda) for t in inputs(R, C, tr, tb))

        def run(res=res, br=br, w=w, gh=gh, go=go):
            hidden, out, rms, kept = mhc.add_rmsnorm_fwd(res, br, w, EPS, 0.2, (1, 2), keep=True)
            return hidden, out, kept.codes, *mhc.add_rmsnorm_bwd(gh, go, hidden, w, rms, 0.2, (1, 2))

        work.append((run, run(), torch.cuda.Stream()))
    torch.cuda.synchronize()

    def repeat(run, want, stream):
        with torch.cuda.stream(stream):
            for _ in range(60):
                got = run()
            if not all(torch.equal(a, b) for a, b in zip(got, want)):
                errors.append("another result")

    threads = [threading.Thread(target=repeat, args=w) for w in work]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not errors


@pytest.mark.gpu
def test_refusals(cuda):
    x, w = torch.randn(4, 16, device=cuda), torch.ones(16, device=cuda)
    with pytest.raises(RuntimeError, match="one shape"):
        mhc.add_rmsnorm(x, x[:1], w)
    with pytest.raises(RuntimeError, match="weight must be 1D"):
        mhc.add_rmsnorm(x, x, w[:8])
    with pytest.raises(RuntimeError, match="float32 or bfloat16"):
        mhc.add_rmsnorm(x, x.half(), w)
    with pytest.raises(RuntimeError, match="needs rng"):
        mhc.add_rmsnorm(x, x, w, 1e-5, 0.1)
    with pytest.raises(RuntimeError, match="eps"):
        mhc.add_rmsnorm(x, x, w, -1.0)
    with pytest.raises(RuntimeError, match="last dimension"):
        mhc.add_rmsnorm(x[:, :0], x[:, :0], w[:0])
    with pytest.raises(RuntimeError, match="codes must be"):
        mhc.add_rmsnorm_quantized(x, x, w, codes=torch.float8_e5m2)
    with pytest.raises(RuntimeError, match="group must be"):
        mhc.add_rmsnorm_quantized(x, x, w, group=64)
    with pytest.raises(RuntimeError, match="no gradient"):
        mhc.add_rmsnorm_quantized(x.clone().requires_grad_(True), x, w)
    h, _, rms, _ = mhc.add_rmsnorm_fwd(x, x, w)
    with pytest.raises(RuntimeError, match="rms must be"):
        mhc.add_rmsnorm_bwd(None, x, h, w, rms[:3])
    with pytest.raises(RuntimeError, match="grad_hidden must have"):
        mhc.add_rmsnorm_bwd(x.bfloat16(), x, h, w, rms)
    with pytest.raises(RuntimeError, match="scales must be"):
        mhc.Coded8(x.to(E4M3), torch.ones(3, device=cuda))
    with pytest.raises(RuntimeError, match="dtype must be"):
        mhc.Coded8(x.to(E4M3), torch.ones(4, 1, device=cuda)).unpack(torch.float16)
    leaf = x.clone().requires_grad_(True)
    hidden, out = mhc.add_rmsnorm(leaf, x, w)
    hidden.detach().add_(1.0)  # the backward pass reads it
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.sum().backward()


@pytest.mark.gpu
@pytest.mark.parametrize("codes", [E4M3, INT8])
@pytest.mark.parametrize("group", [None, 128])
@pytest.mark.parametrize("R,C", [(3, 7), (3, 250), (5, 256), (4, 1000), (3, 1001), (4, 2048), (300, 2048), (2, 4097), (2, 8192),
                                 (300, 8192), (2, 16384), (2, 33000)])
def test_quantized_rows_of_tiny_values(cuda, R, C, group, codes):
    """Rows, and groups of a row, whose scale is the least one, under a reciprocal of the root
    past 2^28: their product is past fp32, the codes are those of the formula all the same."""
    w = torch.ones(C, device=cuda)
    x = torch.zeros(R, C, device=cuda)
    x[1, 0] = 1e-12
    with torch.no_grad():
        for start in (0, 1):  # 1: off alignment, the kernels for any row
            flat = torch.empty(R * C + start, device=cuda)
            v = flat[start:].view(R, C)
            v.copy_(x)
            for eps in (1e-20, 1e-30, 0.0):
                _, q = mhc.add_rmsnorm_quantized(v, torch.zeros_like(v), w, eps, codes, group)
                back = q.unpack(F32)
                if eps:
                    assert not back[0].any() and not back[2:].any()  # NaN counts as one
                assert not back[1, 1:].any()
                want = 1e-12 / ((1e-24 / C) + eps) ** 0.5
                # half a step of e4m3 (2^-4) or int8 at its largest code
                assert back[1, 0].item() == pytest.approx(want, rel=2.0 ** -4)
            # weights below the least scale: 1e-10 / 1e-10 * 1e-30, with h w below fp32's normal values
            v.fill_(1e-10)
            _, q = mhc.add_rmsnorm_quantized(v, torch.zeros_like(v), w * 1e-30, 0.0, codes, group)
            assert bool((q.scales == 2.0 ** -100).all())
            y = 1e-30
            # half a step (of int8 half the scale), and half of h w's last bit, 2^-149 in 1e-40
            tol = y * (2.0 ** -4 + 1e-4) if codes == E4M3 else 2.0 ** -101 + y * 1e-4
            assert bool(((q.unpack(F32).double() - y).abs() <= tol).all())


@pytest.mark.gpu
@pytest.mark.parametrize("R,C", [(200, 256), (200, 250), (2000, 2056), (2000, 2057), (2000, 4096), (2000, 8193)])
def test_weight_gradient_has_a_rounded_reciprocal(cuda, R, C):
    """Row i gives a gradient to column i alone: its sum is 1 / rms of that row, rounded once."""
    R = min(R, C)
    rms = torch.exp(torch.empty(R).uniform_(-7, 7, generator=torch.Generator().manual_seed(C))).to(cuda)
    g = torch.eye(R, C, device=cuda)
    gw = mhc.add_rmsnorm_bwd(None, g, torch.ones(R, C, device=cuda), torch.ones(C, device=cuda), rms)[2]
    want = 1 / rms.double()
    assert bool(((gw[:R].double() - want).abs() <= U * want).all()) and not gw[R:].any()


@pytest.mark.gpu
@pytest.mark.parametrize("tr,tb", [(F32, F32), (F32, BF16), (BF16, F32), (BF16, BF16)])
def test_gradient_of_hidden_alone(cuda, tr, tb):
    """What reaches hidden and not the norm goes through as it is, whatever the row holds."""
    res, br, w, gh, _ = (t.to(cuda) for t in inputs(6, 2056, tr, tb))
    res[0], br[0] = 0.0, 0.0  # without eps its norm has no gradient
    res[1, 5], res[2, 7] = float("inf"), float("nan")
    for p in (0.0, 0.3, 1.0):
        leaves = [t.clone().requires_grad_(True) for t in (res, br, w)]
        hidden, _ = mhc.add_rmsnorm(*leaves, 0.0, p, (3, 4))
        hidden.backward(gh)
        assert torch.equal(leaves[0].grad, gh)
        mask = mhc.dropout_fwd(torch.ones_like(gh, dtype=F32), p, (3, 4))  # 0 or the scale: one product
        assert leaves[1].grad.dtype == tb and torch.equal(leaves[1].grad, (gh.float() * mask).to(tb))
        assert not leaves[2].grad.any()


@pytest.mark.gpu
@pytest.mark.parametrize("tr", [F32, BF16])
@pytest.mark.parametrize("R,C", [(5, 256), (7, 1000), (300, 2048), (4, 2048), (3, 4097), (310, 4104), (300, 8192), (2, 8192),
                                 (3, 9001), (2, 16384)])
def test_dropout_of_a_16_bit_branch(cuda, R, C, tr):
    """Rows that start on alignment: the mask is that of dropout, the product and the sum are
    fp32's, and hidden is rounded once."""
    res, br, w, gh, go = inputs(R, C, tr, BF16)
    p, rng = 0.3, (6, 2 ** 32 - 5)
    keep = mhc.dropout_fwd(torch.ones(R, C, device=cuda), p, rng).cpu() != 0
    scale = 1 / (1 - round(p * 65536) / 65536)
    hidden, out, rms, kept = mhc.add_rmsnorm_fwd(res.to(cuda), br.to(cuda), w.to(cuda), EPS, p, rng, keep=True)
    dropped = torch.where(keep, br.float() * torch.tensor(scale).float(), 0.0)
    assert torch.equal(hidden.cpu(), (res.float() + dropped).to(tr))
    check_out(out.cpu(), hidden.cpu(), w, C, BF16)
    packed = mhc.checkpoint8_pack(out)
    assert torch.equal(kept.codes, packed.codes) and torch.equal(kept.exponents, packed.exponents)
    got = mhc.add_rmsnorm_bwd(gh.to(cuda), go.to(cuda), hidden, w.to(cuda), rms, p, rng)
    check_grads(got, gh, go, hidden.cpu(), w, keep, scale, C, R)
