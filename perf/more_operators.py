"""Performance cases of the operators at the seams and at the end of a step:

* ``dropout``: forward and backward of dropout whose mask comes from a
  counter-based generator and is never stored;
* ``add_norm``: residual addition (with dropout of the branch) and RMSNorm, for
  training (``mode`` train: forward and backward, the normed output also kept in
  8 bits) and for serving (mode e4m3 / int8: the normed output as 8-bit codes
  with fp32 scales);
* ``logprobs``: log probabilities of given tokens with entropy and the most
  likely alternatives, and the gradient of the logits.

The random stream: Philox4x32-10 (Salmon, Moraes, Dror and Shaw, SC 2011) at
counter (offset + g, as two 32-bit words, 0, 0) with the seed's two words as key
gives group g of eight 16-bit numbers, word by word, low half first; value i of a
tensor in row-major order uses number i.  It is dropped where that number is
below t = round(65536 p), and divided by 1 - t / 65536 elsewhere.

hidden = residual + branch is returned in the residual's type, and the norm is of
what is returned.  8-bit codes with scales: a = max |y| over a row or over a group
of 128 columns, scale = max(a / 448, 2^-100) for e4m3 (a / 127 for int8), code =
y / scale rounded to nearest, ties to even.  The kept form of training, of the
output as returned: int8 codes and a power-of-two step for each block of 32 (step
2^e, the smallest e >= -126 with a < 127.5 * 2^e).  Both are returned as the
values that they stand for.

``run`` computes a case in plain torch operations, or, where ``own`` is true,
with this package's operators.  ``exact`` gives the values in 64 bits.
"""
import math

import numpy as np
import torch

own = False

EPS = 1e-5
DT = {"fp32": torch.float32, "bf16": torch.bfloat16}
SIZE = {"fp32": 4, "bf16": 2}
CODE = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}
MOST = {"e4m3": 448.0, "int8": 127.0}
IGNORED = -100
PHILOX_M = (0xD2511F53, 0xCD9E8D57)
PHILOX_W = (0x9E3779B9, 0xBB67AE85)


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------

def listed():
    return [
        # the smallest layer's streams: what counts is the latency
        dict(name="dropout small", op="dropout", R=128, C=256, x="fp32", p=0.1),
        # odd rows and columns
        dict(name="dropout odd", op="dropout", R=1001, C=4097, x="bf16", p=0.3),
        # the streams of the benchmark's training batch (8192 tokens, n = 4, C = 4096)
        dict(name="dropout train", op="dropout", R=32768, C=4096, x="bf16", p=0.1),
        # one token being generated, output in 8 bits for the next product
        dict(name="add_norm token", op="add_norm", R=1, C=4096, res="bf16", x="bf16", mode="e4m3", group=0, p=0.0),
        # a long prompt at the large hidden size, a scale for each 128 columns
        dict(name="add_norm prompt", op="add_norm", R=16384, C=7168, res="bf16", x="bf16", mode="e4m3", group=128, p=0.0),
        # the training batch: 32-bit residual, 16-bit branch with dropout
        dict(name="add_norm train", op="add_norm", R=8192, C=4096, res="fp32", x="bf16", mode="train", group=0, p=0.1),
        # odd sizes in 32 bits
        dict(name="add_norm train odd", op="add_norm", R=1001, C=4097, res="fp32", x="fp32", mode="train", group=0, p=0.0),
        # one generated token with the alternatives that an answer lists
        dict(name="logprobs token", op="logprobs", T=1, V=32768, x="fp32", top=20, grad=False, ignored=0.0, masked=0.0),
        # a batch of generated tokens over a large vocabulary
        dict(name="logprobs batch", op="logprobs", T=64, V=131072, x="fp32", top=20, grad=False, ignored=0.0, masked=0.5),
        # scoring prompts
        dict(name="logprobs score", op="logprobs", T=4096, V=65536, x="bf16", top=5, grad=False, ignored=0.0, masked=0.0),
        # odd vocabulary, masked tokens, padding, 32-bit gradient
        dict(name="logprobs train odd", op="logprobs", T=1001, V=100003, x="fp32", top=0, grad=True, ignored=0.2, masked=0.1),
        # the training batch's loss with an entropy term and its gradient
        dict(name="logprobs train", op="logprobs", T=8192, V=65536, x="bf16", top=0, grad=True, ignored=0.1, masked=0.0),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["dropout", "add_norm", "add_norm", "logprobs", "logprobs"])
    two = lambda: rng.choice(["fp32", "bf16"])  # noqa: E731
    if op == "logprobs":
        V = _log(rng, 32, 131072)
        if rng.random() < 0.6:
            V = max(64, V // 64 * 64)
        T = _log(rng, 1, 32768)
        grad = rng.random() < 0.5
        T = max(1, min(T, (2 ** 28 if grad else 2 ** 27) // V))
        return dict(op=op, T=T, V=V, x=two(), top=rng.choice([0, 1, 5, 20]), grad=grad,
                    ignored=rng.choice([0.0, 0.1, 0.5]), masked=rng.choice([0.0, 0.0, 0.1, 0.4]))
    C = _log(rng, 1, 28672)
    if rng.random() < 0.6:
        C = max(64, C // 64 * 64)
    R = _log(rng, 1, 65536)
    if op == "dropout":
        return dict(op=op, R=max(1, min(R, 2 ** 27 // C)), C=C, x=two(), p=rng.choice([0.05, 0.1, 0.3, 0.5]))
    mode = rng.choice(["train", "train", "e4m3", "int8"])
    group = rng.choice([0, 128]) if mode != "train" else 0
    if group:
        C = max(128, C // 128 * 128)
    R = max(1, min(R, 2 ** 26 // C))
    return dict(op=op, R=R, C=C, res=two(), x=two(), mode=mode, group=group,
                p=rng.choice([0.0, 0.1, 0.3]) if mode == "train" else 0.0)


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) & 0x7FFFFFFF)


def _activations(gen, rows, cols, dtype):
    """Rows of about unit scale with a few loud channels, as residual streams have them."""
    loud = torch.exp(0.5 * torch.randn(cols, device="cuda", generator=gen))
    loud[torch.rand(cols, device="cuda", generator=gen) < 0.002] *= 30.0
    return (torch.randn(rows, cols, device="cuda", generator=gen) * loud).to(dtype)


def prepare(case, seed):
    gen = _gen(seed)
    op, s = case["op"], dict(case)
    rand = lambda *shape: torch.randn(*shape, device="cuda", generator=gen)  # noqa: E731
    if op == "logprobs":
        T, V = case["T"], case["V"]
        # tokens differ in frequency; about half of the rows have one clear answer
        logits = rand(T, V) * 2.0
        logits += torch.randn(V, device="cuda", generator=gen) * 2.0
        rows = torch.arange(T, device="cuda")
        answer = torch.randint(0, V, (T,), device="cuda", generator=gen)
        logits[rows, answer] += 14.0 * torch.rand(T, device="cuda", generator=gen)
        if case["masked"]:  # tokens that are not allowed here; the answer is
            kept = logits[rows, answer].clone()
            logits.masked_fill_(torch.rand(T, V, device="cuda", generator=gen) < case["masked"], -math.inf)
            logits[rows, answer] = kept
        s["logits"] = logits.to(DT[case["x"]])
        other = torch.randint(0, V, (T,), device="cuda", generator=gen)
        given = torch.where((torch.rand(T, device="cuda", generator=gen) < 0.8) | (logits[rows, other] == -math.inf), answer, other)
        s["targets"] = given.masked_fill(torch.rand(T, device="cuda", generator=gen) < case["ignored"], IGNORED)
        if case["grad"]:
            s["grad_logprob"] = -torch.rand(T, device="cuda", generator=gen) / T
            s["grad_entropy"] = rand(T) * 0.01 / T
            if case["top"]:
                s["grad_top"] = rand(T, case["top"]) * 0.1 / T
        return s
    s["rng"] = ((int(seed) * 0x9E3779B97F4A7C15 + 12345) & (2 ** 63 - 1), 8 * int(seed) + 2 ** 33)  # seed, position
    s["x_"] = _activations(gen, case["R"], case["C"], DT[case["x"]])
    if op == "dropout":
        s["grad"] = (rand(case["R"], case["C"]) * 1e-2).to(DT[case["x"]])
        return s
    s["residual"] = _activations(gen, case["R"], case["C"], DT[case["res"]])
    s["weight"] = 0.5 + torch.rand(case["C"], device="cuda", generator=gen)
    if case["mode"] == "train":
        s["grad_hidden"] = (rand(case["R"], case["C"]) * 1e-2).to(DT[case["res"]])
        s["grad_out"] = (rand(case["R"], case["C"]) * 1e-2).to(DT[case["x"]])
    return s


# ---------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------

def _threshold(p):
    return int(round(p * 65536))


def _mask(shape, p, rng):
    """Multiplier of each value: 0, or 1 / (1 - t / 65536) in fp32."""
    count = math.prod(shape)
    groups = (count + 7) // 8
    seed, offset = rng
    low = 0xFFFFFFFF
    at = torch.arange(groups, device="cuda") + offset
    c0, c1 = at & low, (at >> 32) & low
    c2, c3 = torch.zeros_like(c0), torch.zeros_like(c0)
    k0, k1 = seed & low, (seed >> 32) & low
    m0, m1 = PHILOX_M[0] - 2 ** 32, PHILOX_M[1] - 2 ** 32  # as negatives: products stay inside 64 bits
    for _ in range(10):
        hi0, lo0 = ((c0 * m0 >> 32) + c0) & low, (c0 * m0) & low
        hi1, lo1 = ((c2 * m1 >> 32) + c2) & low, (c2 * m1) & low
        c0, c1, c2, c3 = hi1 ^ c1 ^ k0, lo1, hi0 ^ c3 ^ k1, lo0
        k0, k1 = (k0 + PHILOX_W[0]) & low, (k1 + PHILOX_W[1]) & low
    words = torch.stack((c0, c1, c2, c3), 1)
    numbers = torch.stack((words & 0xFFFF, words >> 16), 2).view(-1)[:count]
    t = _threshold(p)
    scale = float(np.float32(1.0 / (1.0 - t / 65536.0)))
    return torch.where(numbers < t, 0.0, scale).view(shape)


def _kept(f):
    """What f [rows, cols] (fp32) stands for after the kept form's 8 bits."""
    rows, cols = f.shape
    f = torch.nn.functional.pad(f, (0, -cols % 32)).view(rows, -1, 32)
    bits = f.abs().amax(-1).view(torch.int32)
    e = (((bits + 0x10000) >> 23) - 6).clamp_(min=1)
    inverse, step = ((254 - e) << 23).view(torch.float32), (e << 23).view(torch.float32)
    return (torch.round(f * inverse.unsqueeze(-1)) * step.unsqueeze(-1)).view(rows, -1)[:, :cols]


def _coded(f, mode, group):
    """What f [rows, cols] (fp32) stands for after 8-bit codes with scales, and the scales."""
    rows, cols = f.shape
    f = f.view(rows, -1, group or cols)
    scales = (f.abs().amax(-1) / MOST[mode]).clamp_(min=2.0 ** -100)
    v = f / scales.unsqueeze(-1)
    v = torch.round(v) if mode == "int8" else v.clamp(-448.0, 448.0).to(torch.float8_e4m3fn).float()
    return (v * scales.unsqueeze(-1)).view(rows, cols), scales


def _top(x, count):
    """(values, indices) of the `count` largest of each row of x (fp32), ties to the lowest index."""
    bits = (x + 0.0).view(torch.int32).long()
    order = torch.where(bits < 0, -(bits & 0x7FFFFFFF), bits)
    index = torch.arange(x.size(1), device=x.device)
    key = (order << 32) + (x.size(1) - 1 - index)
    ids = x.size(1) - 1 - (torch.topk(key, count, dim=1).values & 0xFFFFFFFF)
    return x.gather(1, ids), ids


def _plain_logprobs(s):
    x, t = s["logits"].float(), s["targets"]
    used = t != IGNORED
    at = t.clamp(min=0).unsqueeze(1)
    m = x.amax(1, keepdim=True)
    lse = m + (x - m).exp().sum(1, keepdim=True).log()
    lp = x - lse
    p = lp.exp()
    plogp = torch.where(p > 0, p * lp, 0.0)
    entropy = -plogp.sum(1)
    out = {"logprob": torch.where(used, lp.gather(1, at).squeeze(1), 0.0), "entropy": entropy}
    if s["top"]:
        values, ids = _top(x, s["top"])
        out["top_logprob"], out["top_id"] = values - lse, ids
    if s["grad"]:
        g = torch.where(used, s["grad_logprob"], 0.0).unsqueeze(1)
        total = g.clone()
        if s["top"]:
            total += s["grad_top"].sum(1, keepdim=True)
        gx = -(p * total + (plogp + p * entropy.unsqueeze(1)) * s["grad_entropy"].unsqueeze(1))
        gx.scatter_add_(1, at, g)
        if s["top"]:
            gx.scatter_add_(1, out["top_id"], s["grad_top"])
        out["grad_logits"] = gx.to(s["logits"].dtype)
    return out


def _plain(s):
    if s["op"] == "logprobs":
        return _plain_logprobs(s)
    x = s["x_"].float()
    if s["op"] == "dropout":
        mask = _mask(x.shape, s["p"], s["rng"])
        return {"out": (x * mask).to(s["x_"].dtype), "grad_x": (s["grad"].float() * mask).to(s["x_"].dtype)}
    if s["p"]:
        mask = _mask(x.shape, s["p"], s["rng"])
        x = x * mask
    hidden = (s["residual"].float() + x).to(s["residual"].dtype)
    h, w = hidden.float(), s["weight"]
    rms = torch.sqrt((h * h).mean(1, keepdim=True) + EPS)
    y = h / rms * w
    if s["mode"] != "train":
        values, scales = _coded(y, s["mode"], s["group"])
        return {"hidden": hidden, "out": values.to(torch.bfloat16), "scales": scales}
    out = {"hidden": hidden, "out": y.to(s["x_"].dtype), "kept": _kept(y.to(s["x_"].dtype).float()).to(torch.bfloat16)}
    g = s["grad_out"].float()
    gw = g * w
    dot = (gw * h).sum(1, keepdim=True)
    gi = s["grad_hidden"].float() + (gw - h * (dot / (s["C"] * rms * rms))) / rms
    out["grad_residual"] = gi.to(s["residual"].dtype)
    out["grad_branch"] = (gi * mask if s["p"] else gi).to(s["x_"].dtype)
    out["grad_weight"] = (g * h / rms).sum(0)
    return out


# ---------------------------------------------------------------------------
# the package's operators
# ---------------------------------------------------------------------------

def _own(s):
    import mhc_ascend_b200 as mhc
    if s["op"] == "dropout":
        return {"out": mhc.dropout_fwd(s["x_"], s["p"], s["rng"]), "grad_x": mhc.dropout_fwd(s["grad"], s["p"], s["rng"])}
    if s["op"] == "logprobs":
        got = mhc.token_logprobs_fwd(s["logits"], s["targets"], top=s["top"], ignore_index=IGNORED)
        out = {"logprob": got.logprob, "entropy": got.entropy}
        if s["top"]:
            out["top_logprob"], out["top_id"] = got.top_logprob, got.top_id
        if s["grad"]:
            out["grad_logits"] = mhc.token_logprobs_bwd(s["logits"], s["targets"], got, s["grad_logprob"], s["grad_entropy"],
                                                        s["grad_top"] if s["top"] else None, ignore_index=IGNORED)
        return out
    if s["mode"] != "train":
        hidden, coded = mhc.add_rmsnorm_quantized(s["residual"], s["x_"], s["weight"], EPS, codes=CODE[s["mode"]],
                                                  group=s["group"] or None)
        return {"hidden": hidden, "out": coded.unpack(torch.bfloat16), "scales": coded.scales}
    hidden, y, rms, kept = mhc.add_rmsnorm_fwd(s["residual"], s["x_"], s["weight"], EPS, s["p"], s["rng"], keep=True)
    gr, gb, gw = mhc.add_rmsnorm_bwd(s["grad_hidden"], s["grad_out"], hidden, s["weight"], rms, s["p"], s["rng"])
    return {"hidden": hidden, "out": y, "kept": kept.unpack(torch.bfloat16), "grad_residual": gr, "grad_branch": gb,
            "grad_weight": gw}


def run(state):
    return _own(state) if own else _plain(state)


# ---------------------------------------------------------------------------
# 64 bits, from the definitions
# ---------------------------------------------------------------------------

def _mask64(shape, p, rng):
    """The multipliers again: the generator in unsigned 64-bit integers on the host."""
    count = math.prod(shape)
    position = (np.arange((count + 7) // 8, dtype=np.uint64) + np.uint64(rng[1]))
    word, half = np.uint64(0xFFFFFFFF), np.uint64(32)
    x = [position & word, position >> half, np.zeros_like(position), np.zeros_like(position)]
    key = [rng[0] & 0xFFFFFFFF, (rng[0] >> 32) & 0xFFFFFFFF]
    for _ in range(10):
        a, b = x[0] * np.uint64(PHILOX_M[0]), x[2] * np.uint64(PHILOX_M[1])
        x = [(b >> half) ^ x[1] ^ np.uint64(key[0]), b & word, (a >> half) ^ x[3] ^ np.uint64(key[1]), a & word]
        key = [(key[0] + PHILOX_W[0]) % 2 ** 32, (key[1] + PHILOX_W[1]) % 2 ** 32]
    numbers = np.stack([w.astype(np.uint32) for w in x], axis=1).reshape(-1).astype("<u4").view("<u2")[:count]
    t = _threshold(p)
    return torch.from_numpy(numbers.astype(np.int32) >= t).cuda().double().view(shape) / (1.0 - t / 65536.0)


def _two_to(e):
    """2 ** e in float64, to the bit (a power function may miss by one)."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _kept64(y):
    rows, cols = y.shape
    f = torch.zeros(rows, -(-cols // 32) * 32, dtype=torch.float64, device=y.device)
    f[:, :cols] = y
    f = f.view(rows, -1, 32)
    m, e = torch.frexp(f.abs().amax(-1))  # a = m 2^e, 1/2 <= m < 1
    step = _two_to(torch.where(m < 127.5 / 128.0, e - 7, e - 6).clamp(min=-126)).unsqueeze(-1)
    return (torch.round(f / step) * step).view(rows, -1)[:, :cols]


def _coded64(y, mode, group):
    rows, cols = y.shape
    blocks = y.view(rows, cols // (group or cols), group or cols)
    scales = torch.clamp(blocks.abs().max(-1).values / MOST[mode], min=2.0 ** -100)
    v = blocks / scales[..., None]
    if mode == "int8":
        v = torch.round(v)
    else:  # three bits behind the leading one, steps of 2^-9 at least
        _, e = torch.frexp(v)
        step = _two_to((e - 4).clamp(min=-9))
        v = torch.round(v / step) * step
    return (v * scales[..., None]).view(rows, cols), scales


def _logprobs64(s):
    got = {"logprob": [], "entropy": []}
    if s["top"]:
        got["top_logprob"] = []
    if s["grad"]:
        got["grad_logits"] = torch.empty_like(s["logits"], dtype=torch.float64)
    some = max(1, 2 ** 26 // s["V"])
    for a in range(0, s["T"], some):
        rows = slice(a, a + some)
        logq = torch.log_softmax(s["logits"][rows].double(), 1)
        q = torch.softmax(s["logits"][rows].double(), 1)
        t = s["targets"][rows]
        used = (t >= 0).double()
        one = t.clamp(min=0)
        pick = torch.arange(t.numel(), device=t.device)
        surprise = torch.special.entr(q)  # -q ln q, 0 at 0
        h = surprise.sum(1)
        got["logprob"].append(torch.where(t >= 0, logq[pick, one], 0.0))
        got["entropy"].append(h)
        if s["top"]:
            best, where = torch.sort(s["logits"][rows].float(), dim=1, descending=True, stable=True)
            where = where[:, : s["top"]]
            got["top_logprob"].append(torch.take_along_dim(logq, where, 1))
            del best
        if s["grad"]:
            g = s["grad_logprob"][rows].double() * used
            gt = s["grad_top"][rows].double() if s["top"] else torch.zeros(t.numel(), 1, device=t.device, dtype=torch.float64)
            gx = s["grad_entropy"][rows].double()[:, None] * (surprise - q * h[:, None]) - q * (g + gt.sum(1))[:, None]
            gx[pick, one] += g
            if s["top"]:
                gx.scatter_add_(1, where, gt)
            got["grad_logits"][rows] = gx
    return {k: v if torch.is_tensor(v) else torch.cat(v) for k, v in got.items()}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "logprobs":
        got = _logprobs64(s)
        if case["top"]:
            got["top_id"] = None
        return got
    x = s["x_"].double()
    mask = _mask64(x.shape, case["p"], s["rng"]) if case["p"] else 1.0
    if case["op"] == "dropout":
        return {"out": x * mask, "grad_x": s["grad"].double() * mask}
    h = (s["residual"].double() + x * mask).to(DT[case["res"]]).double()  # the norm is of what is returned
    del x
    w = s["weight"].double()
    r = (h.pow(2).sum(1, keepdim=True) / case["C"] + EPS).sqrt()
    normed = h / r
    if case["mode"] != "train":
        values, scales = _coded64(normed * w, case["mode"], case["group"])
        return {"hidden": h, "out": values, "scales": scales}
    g = s["grad_out"].double()
    projection = (g * w * normed).sum(1, keepdim=True) / case["C"]
    gi = s["grad_hidden"].double() + (g * w - normed * projection) / r
    return {"hidden": h, "out": normed * w, "kept": _kept64((normed * w).to(DT[case["x"]]).double()), "grad_residual": gi, "grad_branch": gi * mask,
            "grad_weight": torch.einsum("rc,rc->c", g, normed)}


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------

def work(case):
    if case["op"] == "logprobs":
        n, e = case["T"] * case["V"], SIZE[case["x"]]
        bytes_ = n * e + case["T"] * (8 + 8 + 12 * case["top"])
        if case["grad"]:
            bytes_ += 2 * n * e + 4 * case["T"] * (2 + case["top"])
        return {"bytes": bytes_, "flops": n * (12 if case["grad"] else 6)}
    n, e = case["R"] * case["C"], SIZE[case["x"]]
    if case["op"] == "dropout":
        return {"bytes": 4 * n * e, "flops": 2 * n}
    h = SIZE[case["res"]]
    if case["mode"] != "train":
        scales = case["R"] * (case["C"] // case["group"] if case["group"] else 1)
        return {"bytes": n * (2 * h + e + 1 + 1 + 2) + 8 * scales + 4 * case["C"], "flops": 6 * n}  # codes written, read, restored
    forward = n * (2 * h + 2 * e + 2 * 33 / 32 + 2)  # codes written, read, restored
    backward = n * (3 * h + 2 * e)  # both incoming gradients and the hidden state; both outgoing ones
    return {"bytes": forward + backward + 12 * case["C"], "flops": 20 * n}
