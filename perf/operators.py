"""Performance cases of the operators around the mHC layer in a training step:

* ``embed`` / ``embed_grad``: token ids -> n residual streams, and the table's
  gradient from the streams' gradient;
* ``pack``: activations stored in 8 bits and restored;
* ``norm``: RMSNorm that keeps its input in 8 bits, forward and backward;
* ``linear_grad``: a linear layer's weight gradient from its input kept in 8
  bits.

The 8-bit form: blocks of 32 along the last dimension; with a = max |x| of the
block, the step is 2^e for the smallest integer e with a < 127.5 * 2^e (e >=
-126), a code is x / 2^e rounded to the nearest integer, ties to even, and
stands for code * 2^e.  Codes are int8 rows padded to a multiple of 128; the
exponents are e + 127 as uint8, one for each 32 codes.

``run`` computes a case in plain torch operations, or, where ``own`` is true,
with this package's operators.  ``exact`` gives the values in 64 bits.
"""
import math

import torch

own = False

BLOCK, PITCH = 32, 128
EPS = 1e-5
DT = {"fp32": torch.float32, "bf16": torch.bfloat16}
SIZE = {"fp32": 4, "bf16": 2}


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------

def listed():
    return [
        # the smallest step: the tests' and the CPU reference's batch
        dict(name="embed small", op="embed", T=32, n=4, C=256, V=32768, table="fp32", out="fp32"),
        # the training batch of the benchmark (8192 tokens, n = 4, C = 4096)
        dict(name="embed train", op="embed", T=8192, n=4, C=4096, V=65536, table="fp32", out="fp32"),
        # the widest rate: 128 tokens, 32 streams of 1280
        dict(name="embed_grad wide", op="embed_grad", T=128, n=32, C=1280, V=32768, table="fp32", out="fp32", pad=0.0),
        # the training batch of the benchmark
        dict(name="embed_grad train", op="embed_grad", T=8192, n=4, C=4096, V=65536, table="fp32", out="fp32", pad=0.0),
        # many tokens in 16 bits, odd sizes, a part of the batch padding
        dict(name="embed_grad long odd", op="embed_grad", T=100003, n=2, C=1281, V=100003, table="bf16", out="bf16", pad=0.2),
        # the smallest layer's streams: what counts is the latency
        dict(name="pack small", op="pack", R=128, C=256, x="fp32"),
        # the streams of the training batch
        dict(name="pack train", op="pack", R=32768, C=4096, x="fp32"),
        # odd rows and columns in 32 bits
        dict(name="norm odd", op="norm", R=1001, C=4097, x="fp32"),
        # a large hidden size in 16 bits
        dict(name="norm wide", op="norm", R=16384, C=7168, x="bf16"),
        # a square projection at the benchmark's width, gradient kept in 32 bits
        dict(name="linear_grad square", op="linear_grad", T=8192, O=4096, K=4096, g="bf16", w="fp32"),
        # 32-bit gradients, odd sizes, few tokens
        dict(name="linear_grad odd fp32", op="linear_grad", T=1001, O=1283, K=1281, g="fp32", w="fp32"),
        # many tokens into the large hidden size, gradient kept in 16 bits
        dict(name="linear_grad long", op="linear_grad", T=32768, O=7168, K=4096, g="bf16", w="bf16"),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["embed", "embed_grad", "pack", "norm", "linear_grad"])
    two = lambda: rng.choice(["fp32", "bf16"])  # noqa: E731
    if op in ("embed", "embed_grad"):
        n = rng.choice([1, 2, 3, 4, 8, 32])
        C = _log(rng, 8, 7168)
        if rng.random() < 0.6:
            C = max(64, C // 64 * 64)
        T = _log(rng, 1, 131072)
        T = max(1, min(T, 8192 * 4 * 4096 // (n * C)))
        V = _log(rng, 100, 131072)
        V = max(2, min(V, 65536 * 4096 // C))
        case = dict(op=op, T=T, n=n, C=C, V=V, table=two(), out=two())
        if op == "embed_grad":
            case["pad"] = rng.choice([0.0, 0.0, 0.1, 0.5])
        return case
    if op in ("pack", "norm"):
        C = _log(rng, 1, 28672)
        if rng.random() < 0.6:
            C = max(64, C // 64 * 64)
        R = _log(rng, 1, 65536)
        R = max(1, min(R, 32768 * 4096 // C))
        return dict(op=op, R=R, C=C, x=two())
    T, O, K = _log(rng, 1, 32768), _log(rng, 8, 8192), _log(rng, 8, 8192)
    if rng.random() < 0.6:
        O, K = max(64, O // 64 * 64), max(64, K // 64 * 64)
    if rng.random() < 0.5:
        T = max(64, T // 64 * 64)
    g = two()
    T = max(1, min(T, 2 ** 39 // (O * K)))
    return dict(op=op, T=T, O=O, K=K, g=g, w=two())


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


def _tokens(gen, count, vocab, pad):
    """Token ids of a text: frequency falls as 1 / rank; a share `pad` is the padding token 0."""
    rank = torch.exp(torch.rand(count, device="cuda", generator=gen) * math.log(vocab)).long().clamp_(1, vocab) - 1
    step = 7919 if vocab % 7919 else 7907
    ids = (rank * step) % vocab
    if pad:
        ids[torch.rand(count, device="cuda", generator=gen) < pad] = 0
    return ids


def _scales(n):
    """The streams' scales: full, then falling."""
    return [0.5 ** i * 8.0 for i in range(n)] if n <= 4 else [1.0 - 0.5 * i / n for i in range(n)]


def prepare(case, seed):
    gen = _gen(seed)
    op, s = case["op"], dict(case)
    rand = lambda *shape: torch.randn(*shape, device="cuda", generator=gen)  # noqa: E731
    if op == "embed":
        s["ids"] = _tokens(gen, case["T"], case["V"], 0.0)
        s["weight"] = (rand(case["V"], case["C"]) * 0.02).to(DT[case["table"]])
        s["scales"] = _scales(case["n"])
    elif op == "embed_grad":
        s["ids"] = _tokens(gen, case["T"], case["V"], case["pad"])
        s["grad"] = (rand(case["T"], case["n"], case["C"]) * 1e-2).to(DT[case["out"]])
        s["scales"] = _scales(case["n"])
    elif op == "pack":
        s["x_"] = _activations(gen, case["R"], case["C"], DT[case["x"]])
    elif op == "norm":
        s["x_"] = _activations(gen, case["R"], case["C"], DT[case["x"]])
        s["weight"] = 0.5 + torch.rand(case["C"], device="cuda", generator=gen)
        s["grad"] = (rand(case["R"], case["C"]) * 1e-2).to(DT[case["x"]])
    else:
        s["codes"], s["exponents"] = _codes(_activations(gen, case["T"], case["K"], torch.bfloat16))
        s["grad"] = (rand(case["T"], case["O"]) * 1e-2).to(DT[case["g"]])
    if "scales" in s:
        s["scales_"] = torch.tensor(s["scales"], device="cuda")
    return s


# ---------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------

def _codes(x):
    """(codes int8 [rows, padded], exponents uint8 [rows, padded / 32]) of x [rows, cols]."""
    rows, cols = x.shape
    wide = (cols + PITCH - 1) // PITCH * PITCH
    f = torch.nn.functional.pad(x.float(), (0, wide - cols)).view(rows, wide // BLOCK, BLOCK)
    bits = f.abs().amax(-1).view(torch.int32)
    e = (((bits + 0x10000) >> 23) - 6).clamp_(min=1)
    inverse = ((254 - e) << 23).view(torch.float32)
    codes = torch.round(f * inverse.unsqueeze(-1)).to(torch.int8).view(rows, wide)
    return codes, e.to(torch.uint8)


def _values(codes, exponents, cols):
    step = (exponents.to(torch.int32) << 23).view(torch.float32)
    f = codes.view(codes.size(0), -1, BLOCK).float() * step.unsqueeze(-1)
    return f.view(codes.size(0), -1)[:, :cols]


def _plain(s):
    op = s["op"]
    if op == "embed":
        scales = s["scales_"]
        rows = s["weight"][s["ids"]].float()
        return (rows.unsqueeze(1) * scales.view(1, -1, 1)).to(DT[s["out"]])
    if op == "embed_grad":
        scales = s["scales_"]
        rows = (s["grad"].float() * scales.view(1, -1, 1)).sum(1)
        if s["pad"]:
            rows = rows * (s["ids"] != 0).unsqueeze(1)
        total = torch.zeros(s["V"], s["C"], device="cuda")
        total.index_add_(0, s["ids"], rows)
        return total.to(DT[s["table"]])
    if op == "pack":
        codes, exponents = _codes(s["x_"])
        return _values(codes, exponents, s["C"]).to(DT[s["x"]])
    if op == "norm":
        x, g, w = s["x_"].float(), s["grad"].float(), s["weight"]
        rms = torch.sqrt((x * x).mean(1, keepdim=True) + EPS)
        out = x / rms * w
        codes, exponents = _codes(s["x_"])
        xh, gw = _values(codes, exponents, s["C"]), g * w
        dot = (gw * xh).sum(1, keepdim=True)
        gx = (gw - xh * (dot / (s["C"] * rms * rms))) / rms
        return {"out": out.to(s["x_"].dtype), "grad_x": gx.to(s["x_"].dtype), "grad_weight": (g * xh / rms).sum(0)}
    xh = _values(s["codes"], s["exponents"], s["K"])
    return (s["grad"].float().t() @ xh).to(DT[s["w"]])


# ---------------------------------------------------------------------------
# the package's operators
# ---------------------------------------------------------------------------

def _own(s):
    import mhc_ascend_b200 as mhc
    op = s["op"]
    if op == "embed":
        return mhc.stream_embedding_fwd(s["ids"], s["weight"], s["n"], s["scales"], dtype=DT[s["out"]])
    if op == "embed_grad":
        return mhc.stream_embedding_bwd(s["grad"], s["ids"], s["V"], s["scales"],
                                        padding_idx=0 if s["pad"] else None, dtype=DT[s["table"]])
    if op == "pack":
        return mhc.checkpoint8_unpack(mhc.checkpoint8_pack(s["x_"]))
    if op == "norm":
        out, rms, kept = mhc.rmsnorm_checkpoint8_fwd(s["x_"], s["weight"], EPS)
        gx, gw = mhc.rmsnorm_checkpoint8_bwd(s["grad"], kept, s["weight"], rms)
        return {"out": out, "grad_x": gx, "grad_weight": gw}
    kept = mhc.Checkpoint8(s["codes"], s["exponents"], (s["T"], s["K"]), torch.bfloat16)
    return mhc.checkpoint8_weight_grad(s["grad"], kept, dtype=DT[s["w"]])


def run(state):
    return _own(state) if own else _plain(state)


# ---------------------------------------------------------------------------
# 64 bits, from the definitions
# ---------------------------------------------------------------------------

def _two_to(e):
    """2 ** e in float64, to the bit (a power function may miss by one)."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _restored64(x):
    """What x [rows, cols] (float64) stands for after 8 bits."""
    rows, cols = x.shape
    count = -(-cols // BLOCK)
    f = torch.zeros(rows, count * BLOCK, dtype=torch.float64, device=x.device)
    f[:, :cols] = x
    f = f.view(rows, count, BLOCK)
    m, e = torch.frexp(f.abs().amax(-1))  # a = m 2^e, 1/2 <= m < 1
    e = torch.where(m < 127.5 / 128.0, e - 7, e - 6)
    step = _two_to(e.clamp(min=-126)).unsqueeze(-1)
    return (torch.round(f / step) * step).view(rows, -1)[:, :cols]


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "embed":
        scales = torch.tensor(s["scales"], device="cuda", dtype=torch.float64)
        out = torch.empty(case["T"], case["n"], case["C"], dtype=torch.float64, device="cuda")
        rows = torch.index_select(s["weight"], 0, s["ids"]).double()
        for i in range(case["n"]):
            torch.mul(rows, scales[i], out=out[:, i])
        return out
    if op == "embed_grad":
        total = torch.zeros(case["V"], case["C"], dtype=torch.float64, device="cuda")
        keep = torch.nonzero(s["ids"] != 0).squeeze(1) if case["pad"] else torch.arange(case["T"], device="cuda")
        for i, scale in enumerate(s["scales"]):
            total.index_add_(0, s["ids"][keep], s["grad"][keep, i].double() * torch.tensor(scale).double().item())
        return total
    if op == "pack":
        return _restored64(s["x_"].double())
    if op == "norm":
        x, g, w = s["x_"].double(), s["grad"].double(), s["weight"].double()
        mean_square = x.pow(2).sum(1, keepdim=True) / case["C"] + EPS
        r = mean_square.sqrt()
        out = w * (x / r)
        del x
        kept = _restored64(s["x_"].double())
        normed = kept / r
        projection = (g * w * normed).sum(1, keepdim=True) / case["C"]
        return {"out": out, "grad_x": (g * w - normed * projection) / r, "grad_weight": torch.einsum("rc,rc->c", g, normed)}
    step = _two_to(s["exponents"].long() - 127)
    kept = (s["codes"].double().view(case["T"], -1, BLOCK) * step.unsqueeze(-1)).view(case["T"], -1)[:, :case["K"]]
    return torch.einsum("to,tk->ok", s["grad"].double(), kept)


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------

def work(case):
    op = case["op"]
    if op == "embed":
        T, n, C = case["T"], case["n"], case["C"]
        rows = min(T, case["V"])
        return {"bytes": 8 * T + rows * C * SIZE[case["table"]] + T * n * C * SIZE[case["out"]], "flops": T * n * C}
    if op == "embed_grad":
        T, n, C = case["T"], case["n"], case["C"]
        live = T * (1.0 - case["pad"])
        return {"bytes": 8 * T + live * n * C * SIZE[case["out"]] + case["V"] * C * SIZE[case["table"]],
                "flops": 2 * live * n * C}
    if op == "pack":
        e = SIZE[case["x"]]
        return {"bytes": case["R"] * case["C"] * (2 * e + 2 * 33 / 32), "flops": 3 * case["R"] * case["C"]}
    if op == "norm":
        e = SIZE[case["x"]]
        return {"bytes": case["R"] * case["C"] * (4 * e + 2 * 33 / 32) + 12 * case["C"] + 8 * case["R"],
                "flops": 14 * case["R"] * case["C"]}
    T, O, K = case["T"], case["O"], case["K"]
    return {"bytes": T * O * SIZE[case["g"]] + T * K * 33 / 32 + O * K * SIZE[case["w"]], "flops": 2 * T * O * K}
