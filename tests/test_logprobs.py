"""Log probabilities of given tokens, entropy, alternatives and the logits'
gradient, against 64 bits."""
import ctypes
import math

import pytest
import torch

import mhc_ascend_b200 as mhc
from mhc_ascend_b200 import _C

U = 2.0 ** -24  # unit roundoff of fp32
UB = 2.0 ** -8  # of bf16
F32, BF16 = torch.float32, torch.bfloat16
INF = float("inf")


def make(T, V, dtype, seed=0, masked=0.0):
    gen = torch.Generator().manual_seed(T * 31 + V + seed)
    x = torch.randn(T, V, generator=gen) * 3
    t = torch.randint(0, V, (T,), generator=gen)
    if masked:
        kept = x.gather(1, t[:, None])
        x[torch.rand(T, V, generator=gen) < masked] = -INF
        x.scatter_(1, t[:, None], kept)
    return x.to(dtype), t


def parts64(x):
    x = x.double()
    m = x.amax(1, keepdim=True)
    d = torch.where(x == -INF, -INF, x - m)
    e = d.exp()
    s = e.sum(1, keepdim=True)
    p = e / s
    far = torch.where(p > 0, -d, 0.0)
    return m, s, p, (p * far).sum(1), (p * far * far).sum(1), far


def slack(V):
    """Additions behind a row's sum (a thread's values, then the trees'), and the few
    roundings of each term: of x - m, its product with log2 e, 2^t (2 units of 2^-23)."""
    return max(64, V // 512) + 24


def check_fwd(got, x, t):
    V = x.size(1)
    m, s, p, e1, e2, _ = parts64(x)
    lp = x.double().gather(1, t.long()[:, None]).squeeze(1) - m.squeeze(1) - s.log().squeeze(1)
    n = slack(V)
    # s: each term off by (3 |x - m| + n) U of itself; then x - m, the logarithm and the difference
    tol = (3 * e1 + n) * U + 3 * U * (lp.abs() + s.log().squeeze(1) + 1)
    err = (got.logprob.double().cpu().flatten() - lp).abs()
    assert bool((err <= tol).all()), f"logprob: max excess {(err - tol).max():.3g}"
    ent = s.log().squeeze(1) + e1
    tol = (3 * e1 + n) * U * (1 + e1) + (3 * e2 + n * e1) * U + 3 * U * (ent + 1)
    err = (got.entropy.double().cpu().flatten() - ent).abs()
    assert bool((err <= tol).all()), f"entropy: max excess {(err - tol).max():.3g}"


def check_top(got, x, k):
    """Ids: those of a stable sort, largest first (zeros equal)."""
    f = x.float() + 0.0
    order = torch.sort(f, dim=1, descending=True, stable=True).indices[:, :k]
    ids = got.top_id.cpu().view(-1, k)
    assert torch.equal(ids, order), f"{(ids != order).sum()} ids differ"
    m, s, _, e1, _, _ = parts64(x)
    lp = f.double().gather(1, ids) - m - s.log()
    val = got.top_logprob.double().cpu().view(-1, k)
    assert torch.equal(torch.isinf(val), torch.isinf(lp))
    fin = torch.isfinite(lp)
    tol = ((3 * e1 + slack(x.size(1))) * U)[:, None] + 3 * U * (lp.abs() + s.log() + 1)
    assert bool(((val - lp).abs() <= tol)[fin].all())


# ---------------------------------------------------------------------------
# no GPU needed
# ---------------------------------------------------------------------------

def test_cpu_tensors_raise():
    with pytest.raises(RuntimeError, match="CUDA"):
        mhc.token_logprobs(torch.randn(2, 8), torch.zeros(2, dtype=torch.int64))


def test_entry_points_validate_without_gpu():
    lib = _C.load()
    p, odd = ctypes.c_void_p(16), ctypes.c_void_p(18)

    def fwd(x=p, t=p, lp=p, ent=p, tv=None, ti=None, st=p, T=4, V=64, stride=64, top=0, bf16=0):
        return lib.mhc_token_logprobs_fwd(x, bf16, stride, t, 1, -100, lp, ent, tv, ti, st, T, V, top, None)

    assert fwd(T=0) == 0
    assert fwd(T=-1) == -1 and fwd(V=0, stride=1) == -1 and fwd(stride=63) == -1 and "row_stride" in _C.last_error()
    assert fwd(x=None) == -1 and fwd(t=None) == -1 and fwd(lp=None) == -1 and fwd(ent=None) == -1 and fwd(st=None) == -1
    assert fwd(top=33) == -2 and fwd(top=-1) == -2 and fwd(V=8, stride=8, top=9) == -2 and "min(32" in _C.last_error()
    assert fwd(top=4) == -1 and fwd(top=4, tv=p) == -1
    assert fwd(V=(1 << 21) + 1, stride=1 << 22) == -2 and fwd(T=1 << 31) == -2
    assert fwd(x=odd) == -3

    def bwd(x=p, gx=p, st=p, ent=p, ids=None, gt=None, T=4, V=64, top=0):
        return lib.mhc_token_logprobs_bwd(x, 0, 64, p, 0, -100, st, ent, ids, p, None, gt, gx, T, V, top, None)

    assert bwd(T=0) == 0 and bwd(x=None) == -1 and bwd(gx=None) == -1 and bwd(st=None) == -1 and bwd(ent=None) == -1
    assert bwd(top=2) == -1 and bwd(top=2, ids=p) == -1 and bwd(top=40) == -2


# ---------------------------------------------------------------------------
# GPU: forward
# ---------------------------------------------------------------------------

SIZES = [(1, 1), (3, 2), (2, 5), (4, 7), (5, 8), (3, 31), (40, 33), (300, 195), (7, 256), (2, 1000), (1, 4099), (3, 8191),
         (2, 8200), (1, 32768), (320, 8300), (300, 20001), (5, 32771), (1, 100003), (3, 131072), (150, 65536), (700, 16640),
         (1, 1 << 21), (2, (1 << 21) - 1), (100, 262147)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("T,V", SIZES)
def test_forward(cuda, T, V, dtype):
    x, t = make(T, V, dtype)
    t = t.int() if T % 2 else t
    k = min(V, 32 if T < 10 else 5)
    for top in (0, 1, k):
        got = mhc.token_logprobs(x.to(cuda), t.to(cuda), top)
        assert got.logprob.shape == (T,) and got.logprob.dtype == F32
        check_fwd(got, x, t)
        if top:
            check_top(got, x, top)
        else:
            assert got.top_id is None and got.top_logprob is None


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("T,V", [(1, 300), (2, 8200), (400, 5000), (1, 65537), (300, 9000)])
@pytest.mark.parametrize("kind", ["ties", "equal", "rising", "falling", "few", "zeros", "lowest", "one segment", "last"])
def test_alternatives_in_hard_orders(cuda, T, V, dtype, kind):
    gen = torch.Generator().manual_seed(V)
    if kind == "ties":
        x = torch.randint(0, 4, (T, V), generator=gen).float()
    elif kind == "equal":
        x = torch.full((T, V), 1.5)
    elif kind in ("rising", "falling"):
        x = torch.linspace(-8, 8, V).expand(T, V).clone()
        x = x.flip(1) if kind == "falling" else x
    elif kind == "few":  # fewer possible tokens than alternatives
        x = torch.full((T, V), -INF)
        x[:, V // 3], x[:, V - 1], x[:, 0] = 1.0, 2.0, 1.0
    elif kind == "zeros":  # +0 and -0 are equal
        x = torch.zeros(T, V)
        x[:, ::2] = -0.0
    elif kind == "lowest":  # masks of the type's lowest value
        x = torch.full((T, V), torch.finfo(dtype).min)
        x[:, 5:9] = torch.tensor([0.5, 0.25, 0.75, -3.0])
    elif kind == "one segment":  # all of the largest next to each other
        x = torch.randn(T, V, generator=gen)
        x[:, 100:164] = torch.linspace(20, 30, 64)
    else:
        x = torch.randn(T, V, generator=gen)
        x[:, -40:] += 50
    x = x.to(dtype)
    t = torch.zeros(T, dtype=torch.int64)
    got = mhc.token_logprobs(x.to(cuda), t.to(cuda), 20)
    check_top(got, x, 20)
    check_fwd(got, x, t)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("T,V", [(1, 40000), (500, 3001)])
def test_masked(cuda, T, V, dtype):
    x, t = make(T, V, dtype, masked=0.5)
    got = mhc.token_logprobs(x.to(cuda), t.to(cuda), 10)
    check_fwd(got, x, t)
    check_top(got, x, 10)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("V", [64, 9001, 40000])
def test_rows_without_a_distribution(cuda, V, dtype):
    x = torch.randn(6, V).to(dtype)
    x[0] = -INF
    x[1, V // 2] = INF
    x[2, 7] = float("nan")
    x[3] = torch.finfo(dtype).min
    x[4, :] = -INF
    x[4, 3] = -5.0
    t = torch.tensor([3, 3, 3, 3, 3, 3])
    for top in (0, 4):
        leaf = x.to(cuda).requires_grad_(True)
        got = mhc.token_logprobs(leaf, t.to(cuda), top)
        lp, ent = got.logprob.tolist(), got.entropy.tolist()
        assert lp[0] == -INF and ent[0] == 0.0
        assert math.isnan(lp[1]) and math.isnan(ent[1]) and math.isnan(lp[2]) and math.isnan(ent[2])
        # V equal logits: V exact ones, added in fp32
        assert lp[3] == pytest.approx(-math.log(V), rel=4 * U) and ent[3] == pytest.approx(math.log(V), rel=4 * U)
        assert lp[4] == 0.0 and ent[4] == 0.0
        if top:
            assert (got.top_logprob[0] == -INF).all() and got.top_id[0].tolist() == [0, 1, 2, 3]
            assert got.top_id[3].tolist() == [0, 1, 2, 3] and got.top_id[4].tolist() == [3, 0, 1, 2]
            assert torch.isnan(got.top_logprob[1:3]).all() and got.top_id[1, 0] == V // 2
        (got.logprob.sum() + got.entropy.sum()).backward()
        g = leaf.grad.float()
        assert not g[0].any() and torch.isnan(g[1]).all() and torch.isnan(g[2]).all()
        assert torch.isfinite(g[3:]).all() and not g[4].any()
    every = torch.full((2, V), float("nan"), device=cuda, dtype=dtype)
    got = mhc.token_logprobs(every, t[:2].to(cuda), 3)
    assert torch.isnan(got.logprob).all() and got.top_id.tolist() == [[0, 1, 2]] * 2


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("T,V", [(1, 40000), (2, 70), (300, 9001)])
@pytest.mark.parametrize("most", [3e38, 1.5e38, 2e37, 5e36, -5e36, -2e37, -1.5e38, -3e38])
def test_logits_next_to_overflow(cuda, T, V, dtype, most):
    """Rows whose maximum is huge, with masked and far smaller logits beside it."""
    x = torch.full((T, V), most)
    x[:, V // 2:] = -INF
    x[:, 0], x[:, 1], x[:, V - 1] = torch.finfo(dtype).min, 0.0 if most > 0 else most * 1.1, most
    x = x.to(dtype)
    t = torch.full((T,), V - 1)
    count = int((x[0] == x[0].max()).sum())  # all others are infinitely far
    got = mhc.token_logprobs(x.to(cuda).requires_grad_(True), t.to(cuda), 4)
    assert got.logprob[0].item() == pytest.approx(-math.log(count), rel=4 * U, abs=2 * U)
    assert got.entropy[0].item() == pytest.approx(math.log(count), rel=4 * U, abs=2 * U)
    assert torch.equal(got.logprob, got.logprob[:1].expand(T))
    order = torch.sort(x.float(), dim=1, descending=True, stable=True).indices[:, :4]
    assert torch.equal(got.top_id.cpu(), order)
    r = mhc.token_logprobs_fwd(x.to(cuda), t.to(cuda))
    one = torch.ones(T, device=cuda)
    gx = mhc.token_logprobs_bwd(x.to(cuda), t.to(cuda), r, one, one).double().cpu()
    p = (x == x[0].max()).double() / count  # log p and the entropy cancel: the gradient is the logprob's alone
    want = -p
    want[:, V - 1] += 1
    # rounded once to its type: half a step of the value (1 - p of the given token is not exact in 24 bits); p by a few units
    assert bool(((gx - want).abs() <= (UB if dtype == BF16 else U) * want.abs() + 64 * U * p).all())


@pytest.mark.gpu
def test_targets_outside(cuda):
    x, _ = make(5, 100, F32)
    t = torch.tensor([-100, 100, -1, 1 << 40, 99])
    leaf = x.to(cuda).requires_grad_(True)
    got = mhc.token_logprobs(leaf, t.to(cuda))
    assert got.logprob[0] == 0 and torch.isnan(got.logprob[1:4]).all() and torch.isfinite(got.logprob[4])
    check_fwd(mhc.TokenLogprobs(got.logprob[4:], got.entropy[4:], None, None), x[4:], t[4:])
    got.logprob[torch.isfinite(got.logprob)].sum().backward()
    assert not leaf.grad[0].any() and leaf.grad[4].any()
    (g,) = torch.autograd.grad(mhc.token_logprobs(leaf, t.to(cuda)).logprob.sum(), leaf)
    assert torch.isnan(g[1:4]).all() and not g[0].any()
    inside = mhc.token_logprobs(leaf, torch.tensor([7] * 5, device=cuda), ignore_index=7)
    assert not inside.logprob.any()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_layouts(cuda, dtype):
    x, t = make(24, 1003, dtype)
    want = mhc.token_logprobs(x.to(cuda), t.to(cuda), 7)
    wide = torch.zeros(24, 1203, device=cuda, dtype=dtype)
    for off in (1, 2, 5, 8):
        wide[:, off:off + 1003] = x.to(cuda)
        view = wide[:, off:off + 1003]
        got = mhc.token_logprobs(view, t.to(cuda), 7)
        assert torch.equal(got.top_id, want.top_id)
        check_fwd(got, x, t)
        g = torch.randn(24, device=cuda)
        r = mhc.token_logprobs_fwd(view, t.to(cuda))
        check_grad(mhc.token_logprobs_bwd(view, t.to(cuda), r, g, g), x, t, g.cpu(), g.cpu(), None, None)
    got = mhc.token_logprobs(x.to(cuda).view(2, 3, 4, 1003), t.to(cuda).view(2, 3, 4), 7)
    assert got.logprob.shape == (2, 3, 4) and got.top_id.shape == (2, 3, 4, 7)
    assert torch.equal(got.logprob.flatten(), want.logprob)
    one = mhc.token_logprobs(x[0].to(cuda), t[0].to(cuda), 7)
    assert one.logprob.shape == () and one.top_id.shape == (7,)
    turned = mhc.token_logprobs(x.to(cuda).t().contiguous().t(), t.to(cuda), 7)
    assert torch.equal(turned.logprob, want.logprob)
    none = mhc.token_logprobs(x[:0].to(cuda), t[:0].to(cuda), 7)
    assert none.logprob.shape == (0,) and none.top_id.shape == (0, 7)
    rows = mhc.token_logprobs(x[:1].to(cuda).expand(24, 1003), t[:1].to(cuda).expand(24), 7)
    assert torch.equal(rows.entropy, rows.entropy[:1].expand(24))


@pytest.mark.gpu
def test_rows_past_32_bits(cuda):
    T, V = 70000, 65536  # 4.6e9 logits
    x = torch.zeros(T, V, device=cuda, dtype=BF16)
    x[-1] = torch.linspace(-4, 4, V).to(BF16).to(cuda)
    x[T // 2, 17] = 30.0
    t = torch.full((T,), 17, device=cuda)
    got = mhc.token_logprobs_fwd(x, t, 3)
    check_fwd(mhc.TokenLogprobs(got.logprob[-1:], got.entropy[-1:], None, None), x[-1:].cpu(), t[-1:].cpu())
    assert got.top_id[T // 2].tolist() == [17, 0, 1] and got.top_id[-1, 0] >= V - 512
    assert bool((got.logprob[:100] + math.log(V)).abs().max() < 1e-5)
    g = torch.ones(T, device=cuda)
    gx = mhc.token_logprobs_bwd(x, t, got, g)
    for row in (0, T // 2, T - 1):
        check_grad(gx[row:row + 1], x[row:row + 1].cpu(), t[:1].cpu(), g[:1].cpu(), None, None, None)


# ---------------------------------------------------------------------------
# GPU: gradient
# ---------------------------------------------------------------------------

def check_grad(gx, x, t, gl, ge, gt, ids):
    T, V = x.shape
    m, s, p, e1, e2, far = parts64(x)
    ent = s.log() + e1[:, None]
    lnp = -far - s.log()
    zero = torch.zeros(T, dtype=torch.float64)
    gl = zero if gl is None else torch.where(t >= 0, gl.double(), 0.0)
    ge = zero if ge is None else ge.double()
    own, own_mag = torch.zeros(T, V, dtype=torch.float64), torch.zeros(T, V, dtype=torch.float64)
    at = t.long().clamp(min=0)[:, None]
    own.scatter_add_(1, at, gl[:, None])
    own_mag.scatter_add_(1, at, gl.abs()[:, None])
    G, Gm = gl.clone(), gl.abs()
    if gt is not None:
        own.scatter_add_(1, ids, gt.double())
        own_mag.scatter_add_(1, ids, gt.double().abs())
        G, Gm = G + gt.double().sum(1), Gm + gt.double().abs().sum(1)
    want = own - p * (G[:, None] + ge[:, None] * (lnp + ent))
    n = slack(V)
    # p as in the forward, twice (2^t and s); the bracket's terms each off by a few units, the entropy as in the forward
    brack = Gm[:, None] + ge.abs()[:, None] * (far + 2 * s.log() + ent)
    off = (3 * far + 3 * e1[:, None] + 2 * n) * U
    ent_off = ((3 * e1 + n) * U * (1 + e1) + (3 * e2 + n * e1) * U + 3 * U * (ent.squeeze(1) + 1))[:, None]
    tol = p * (off * brack + (40 + n) * U * brack + ge.abs()[:, None] * ent_off) + 40 * U * own_mag + 1e-38
    tol = tol + (UB if gx.dtype == BF16 else U) * want.abs() * (1 + UB) + (2.0 ** -133 if gx.dtype == BF16 else 0)
    err = (gx.double().cpu().view(T, V) - want).abs()
    assert bool((err <= tol).all()), f"gradient: max excess {(err - tol).max():.3g}"


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("T,V", [(1, 1), (3, 2), (5, 7), (40, 33), (30, 195), (7, 256), (4, 4099), (3, 8200), (2, 32771),
                                 (6, 20001), (2, 100003), (300, 1000)])
def test_gradient(cuda, T, V, dtype):
    x, t = make(T, V, dtype, masked=0.3 if V > 30 else 0.0)
    t[::3] = -100
    gen = torch.Generator().manual_seed(V)
    k = min(V, 6)
    gl, ge, gt = torch.randn(T, generator=gen), torch.randn(T, generator=gen), torch.randn(T, k, generator=gen)
    r = mhc.token_logprobs_fwd(x.to(cuda), t.to(cuda), k)
    r0 = mhc.token_logprobs_fwd(x.to(cuda), t.to(cuda))
    for a, b, c in ((gl, None, None), (None, ge, None), (gl, ge, None), (gl, ge, gt), (None, None, gt), (None, None, None)):
        dev = [None if g is None else g.to(cuda) for g in (a, b, c)]
        gx = mhc.token_logprobs_bwd(x.to(cuda), t.to(cuda), r, *dev)
        assert gx.dtype == dtype and gx.shape == (T, V)
        check_grad(gx, x, t, a, b, c, r.top_id.cpu())
        if c is None:
            assert torch.equal(gx, mhc.token_logprobs_bwd(x.to(cuda), t.to(cuda), r0, *dev))


@pytest.mark.gpu
def test_autograd_against_differences(cuda):
    T, V, k = 4, 50, 3
    x, t = make(T, V, F32)
    t[1] = -100
    x[2, 4:9] = -INF
    leaf = x.to(cuda).requires_grad_(True)
    got = mhc.token_logprobs(leaf, t.to(cuda), k)
    gen = torch.Generator().manual_seed(1)
    a, b, c = torch.randn(T, generator=gen), torch.randn(T, generator=gen), torch.randn(T, k, generator=gen)
    ((got.logprob * a.to(cuda)).sum() + (got.entropy * b.to(cuda)).sum() + (got.top_logprob * c.to(cuda)).sum()).backward()
    ids = got.top_id.cpu()

    def loss(x):
        # -inf as -1000, of probability 0 in 64 bits too: a masked target's log probability then has differences
        q = torch.log_softmax(x, 1)
        ent = torch.special.entr(q.exp()).sum(1)
        lp = torch.where(t >= 0, q.gather(1, t.clamp(min=0)[:, None]).squeeze(1), 0.0)
        return ((lp * a.double()).sum() + (ent * b.double()).sum() + (q.gather(1, ids) * c.double()).sum()).item()

    step, finite = 1e-5, x.double().nan_to_num(neginf=-1000.0)
    for _ in range(5):
        d = torch.randn(T, V, generator=gen, dtype=torch.float64)
        slope = (loss(finite + step * d) - loss(finite - step * d)) / (2 * step)
        got_slope = (leaf.grad.cpu().double() * d).sum().item()
        # third derivatives of size ~10 for each of 4 rows x step^2; gradients of size ~3 off by ~100 U, 200 of them
        assert got_slope == pytest.approx(slope, abs=4 * 100 * step ** 2 + 200 * 3 * 100 * U + 1e-6)


@pytest.mark.gpu
def test_autograd_parts(cuda):
    x, t = make(9, 300, BF16)
    leaf = x.to(cuda).requires_grad_(True)
    got = mhc.token_logprobs(leaf, t.to(cuda), 2)
    assert not got.top_id.requires_grad and got.top_logprob.requires_grad
    (g,) = torch.autograd.grad(-got.logprob.mean(), leaf)
    gl = torch.full((9,), -1.0 / 9, device=cuda)
    r = mhc.token_logprobs_fwd(leaf.detach(), t.to(cuda))
    assert torch.equal(g, mhc.token_logprobs_bwd(leaf.detach(), t.to(cuda), r, gl))
    best = mhc.token_logprobs(leaf, t.to(cuda), 2)
    (g,) = torch.autograd.grad(best.top_logprob[:, 0].sum(), leaf)
    one = mhc.token_logprobs(leaf, best.top_id[:, 0])
    (h,) = torch.autograd.grad(one.logprob.sum(), leaf)
    assert torch.equal(g, h)
    with torch.no_grad():
        assert not mhc.token_logprobs(leaf, t.to(cuda)).logprob.requires_grad


@pytest.mark.gpu
def test_captured_on_another_stream(cuda):
    x, t = (v.to(cuda) for v in make(12, 30001, BF16))
    g = torch.randn(12, device=cuda)

    def step():
        r = mhc.token_logprobs_fwd(x, t, 5)
        return r.logprob, r.entropy, r.top_logprob, r.top_id, mhc.token_logprobs_bwd(x, t, r, g, g)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        want = step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for v in got:
        v.zero_()
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    x2, t2 = make(12, 30001, BF16, seed=9)
    x.copy_(x2), t.copy_(t2)
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(got, step()))


@pytest.mark.gpu
def test_refusals(cuda):
    x, t = torch.randn(3, 20, device=cuda), torch.zeros(3, dtype=torch.int64, device=cuda)
    for bad, what in ((dict(logits=x.half()), "float32 or bfloat16"), (dict(targets=t.float()), "int64 or int32"),
                      (dict(targets=t[:2]), "leading dimensions"), (dict(top=21), "top must be"), (dict(top=-1), "top must be"),
                      (dict(logits=x[:, :0]), "vocabulary"), (dict(targets=t.cpu()), "CUDA")):
        with pytest.raises(RuntimeError, match=what):
            mhc.token_logprobs(**{"logits": x, "targets": t, **bad})
    r = mhc.token_logprobs_fwd(x, t, 2)
    with pytest.raises(RuntimeError, match="grad_top must have"):
        mhc.token_logprobs_bwd(x, t, r, None, None, torch.ones(3, 3, device=cuda))
    with pytest.raises(RuntimeError, match="targets' shape"):
        mhc.token_logprobs_bwd(x, t, r, torch.ones(2, device=cuda))
    with pytest.raises(RuntimeError, match="for these logits"):
        mhc.token_logprobs_bwd(x, t, mhc.token_logprobs_fwd(x[:2], t[:2]), None)
    for bad in (r._replace(stats=r.stats.cpu()), r._replace(entropy=r.entropy.cpu()), r._replace(top_id=r.top_id.cpu())):
        with pytest.raises(RuntimeError, match="CUDA"):
            mhc.token_logprobs_bwd(x, t, bad, None, None, torch.ones(3, 2, device=cuda))
    with pytest.raises(RuntimeError, match="for these logits"):
        mhc.token_logprobs_bwd(x, t, r._replace(top_id=r.top_id.int()), None, None, torch.ones(3, 2, device=cuda))
    with pytest.raises(RuntimeError, match="at most"):
        mhc.token_logprobs(torch.empty(1, (1 << 21) + 1, device=cuda), t[:1])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("mask", ["-inf", "lowest"])
@pytest.mark.parametrize("T,V", [(5, 200), (3, 1003), (2, 40000), (300, 9000)])
def test_entropy_gradients_over_masked_logits(cuda, T, V, dtype, mask):
    """Confident rows (a sum of exponentials of about 1) under entropy gradients above it."""
    x, t = make(T, V, dtype, seed=5)
    x[:, 3] = 30.0
    x[:, V // 4:V // 2] = -INF if mask == "-inf" else torch.finfo(dtype).min
    t[:] = V - 1
    gl = torch.randn(T, generator=torch.Generator().manual_seed(V))
    r = mhc.token_logprobs_fwd(x.to(cuda), t.to(cuda))
    for size in (2.0, 3.0, 1e3, 65536.0, 1e30):
        for sign in (1, -1):
            ge = torch.full((T,), sign * size)
            for a in (None, gl):
                gx = mhc.token_logprobs_bwd(x.to(cuda), t.to(cuda), r, None if a is None else a.to(cuda), ge.to(cuda))
                assert not gx[:, V // 4:V // 2].any()  # NaN counts as one
                check_grad(gx, x, t, a, ge, None, None)
    for loss in (lambda e: 3 * e.sum(), lambda e: (e + 5).exp().sum()):
        leaf = x.to(cuda).requires_grad_(True)
        loss(mhc.token_logprobs(leaf, t.to(cuda)).entropy).backward()
        assert torch.isfinite(leaf.grad).all()


@pytest.mark.gpu
@pytest.mark.parametrize("V", [100, 9001])
def test_targets_outside_touch_the_log_probability_alone(cuda, V):
    """Entropies and alternatives do not depend on the target, nor do their gradients."""
    x, _ = make(4, V, F32)
    t = torch.tensor([-1, V, 1 << 40, 5]).to(cuda)
    r = mhc.token_logprobs_fwd(x.to(cuda), t, 3)
    gen = torch.Generator().manual_seed(1)
    ge, gt = torch.randn(4, generator=gen), torch.randn(4, 3, generator=gen)
    zero = torch.zeros(4, dtype=torch.int64)
    for a, b in ((ge, None), (None, gt), (ge, gt)):
        dev = [None if g is None else g.to(cuda) for g in (a, b)]
        check_grad(mhc.token_logprobs_bwd(x.to(cuda), t, r, None, *dev), x, zero, None, a, b, r.top_id.cpu())
    gx = mhc.token_logprobs_bwd(x.to(cuda), t, r, ge.to(cuda))
    assert torch.isnan(gx[:3]).all() and torch.isfinite(gx[3]).all()
    leaf = x.to(cuda).requires_grad_(True)
    mhc.token_logprobs(leaf, t).entropy.sum().backward()
    assert torch.isfinite(leaf.grad).all()
