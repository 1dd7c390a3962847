"""The operators of a step together, as a model uses them: streams in, blocks with
dropout, plain residual and norm, linear layers from 8 bits, log probabilities out."""
import importlib.util
import os

import pytest
import torch

import mhc_ascend_b200 as mhc
from mhc_ascend_b200.ops import stream_mean

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def parameters(cuda, V=300, C=96, n=4):
    gen = torch.Generator().manual_seed(3)
    rand = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    p = [rand(V, C), rand(2 * C, C) * C ** -0.5, rand(C, 2 * C) * (2 * C) ** -0.5, 0.5 + torch.rand(C, generator=gen),
         0.5 + torch.rand(C, generator=gen), rand(V, C) * C ** -0.5]
    ids = torch.randint(1, V, (40,), generator=gen)
    ids[-5:] = 0
    return [t.to(cuda) for t in p], ids.to(cuda)


def step(params, ids, rng, p, eight, top=0):
    """Logits' results of one small model: embedding, mean, norm, a branch, residual and
    norm, head.  eight: the 8-bit operators; otherwise plain torch with the same mask."""
    table, up, down, w1, w2, head = params
    C = table.size(1)
    if eight:
        h = stream_mean(mhc.stream_embedding(ids[:-1], table, 4, [1.0, 0.5, 0.25, 0.125], padding_idx=0))
        y = mhc.rmsnorm(h, w1)
        branch = mhc.linear_checkpoint8(torch.relu(mhc.linear_checkpoint8(y, up)), down)
        hidden, out, kept = mhc.add_rmsnorm(h, branch, w2, 1e-5, p, rng, keep=True)
        logits = mhc.linear_checkpoint8(out, head, kept=kept)
        return mhc.token_logprobs(logits, ids[1:], top, ignore_index=0), hidden
    h = torch.nn.functional.embedding(ids[:-1], table, padding_idx=0) * 0.46875
    norm = lambda t, w: t / (t.square().mean(-1, keepdim=True) + 1e-5).sqrt() * w  # noqa: E731
    branch = torch.relu(norm(h, w1) @ up.t()) @ down.t()
    mask = mhc.dropout_fwd(torch.ones(branch.shape, device=ids.device), p, rng).double()
    hidden = h + branch * mask
    q = torch.log_softmax(norm(hidden, w2) @ head.t(), -1)
    lp = torch.where(ids[1:] != 0, q.gather(1, ids[1:, None]).squeeze(1), 0.0)
    return (lp, torch.special.entr(q.exp()).sum(-1), q), hidden


def test_step_and_gradients(cuda):
    params, ids = parameters(cuda)
    counter = mhc.DropoutCounter(5).to(cuda)
    rng = counter.take(mhc.dropout_groups((39, 96)))
    leaves = [t.clone().requires_grad_(True) for t in params]
    got, hidden = step(leaves, ids, rng, 0.2, True, top=3)
    counter.take(10)  # the next step's numbers do not touch this one's backward pass
    (-got.logprob.sum() + 0.1 * got.entropy.sum() + 1e-3 * hidden.square().sum()).backward()
    exact = [t.double().requires_grad_(True) for t in params]
    (lp, ent, q), hid = step(exact, ids, rng, 0.2, False)
    (-lp.sum() + 0.1 * ent.sum() + 1e-3 * hid.square().sum()).backward()
    # the forward pass is the same formulas in fp32: a few hundred roundings behind each value
    assert (got.logprob.double() - lp).abs().max() < 1000 * U * lp.abs().max()
    assert (got.entropy.double() - ent).abs().max() < 1000 * U * ent.abs().max()
    assert torch.equal(got.top_id, torch.topk(q, 3).indices)
    # the weights of the linear layers take their inputs from 8 bits: 0.6% of their rms for
    # each term, which do not add up over tokens; the others come from the same formulas
    for a, e, tol in zip(leaves, exact, (1e-4, 0.02, 0.02, 1e-4, 1e-4, 0.02)):
        err = (a.grad.double() - e.grad).norm() / e.grad.norm()
        assert err < tol, f"{tuple(a.shape)}: {err:.3g}"
    assert not leaves[0].grad[0].any()


def test_captured_step(cuda):
    """A whole step with its backward pass in a graph: new numbers each time it is replayed."""
    params, ids = parameters(cuda)
    leaves = [t.clone().requires_grad_(True) for t in params]
    counter = mhc.DropoutCounter(5).to(cuda)
    groups = mhc.dropout_groups((39, 96))

    def run():
        got, _ = step(leaves, ids, counter.take(groups), 0.2, True)
        return (got.logprob.detach(), *torch.autograd.grad(-got.logprob.sum(), leaves))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(3):
            run()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = run()
    seen = []
    for turn in range(3):
        graph.replay()
        seen.append([t.clone() for t in held])
    assert counter.state[1].item() == 6 * groups
    for turn in range(3):
        counter.state[1] = (3 + turn) * groups
        assert torch.equal(run()[0], seen[turn][0])
    assert not torch.equal(seen[0][0], seen[1][0])


def test_serving_step(cuda):
    """One token after another: residual, 8-bit norm output, head, alternatives."""
    params, ids = parameters(cuda)
    with torch.no_grad():
        residual = params[0][ids[:4]].bfloat16()
        branch = torch.randn(4, 96, device=cuda).bfloat16()
        every, q = mhc.add_rmsnorm_quantized(residual, branch, params[4])
        logits = q.unpack() @ params[5].t().bfloat16()
        whole = mhc.token_logprobs(logits, ids[1:5], top=5)
        for i in range(4):
            hidden, q1 = mhc.add_rmsnorm_quantized(residual[i:i + 1], branch[i:i + 1], params[4])
            assert torch.equal(hidden, every[i:i + 1]) and torch.equal(q1.codes.view(torch.uint8), q.codes[i:i + 1].view(torch.uint8))
            one = mhc.token_logprobs(logits[i], ids[i + 1], top=5)
            assert torch.equal(one.top_id, whole.top_id[i]) and torch.equal(one.logprob, whole.logprob[i])


@pytest.mark.parametrize("mode", ["fused", "kept", "packed"])
def test_wrapper_with_branch_dropout(cuda, mode):
    kw = dict(checkpoint_8bit=mode == "kept")
    n = 2 if mode == "packed" else 4
    torch.manual_seed(0)
    drops = mhc.MHCResidualWrapper(128, n, branch_dropout=0.25, dropout_seed=11, **kw).to(cuda)
    plain = mhc.MHCResidualWrapper(128, n, **kw).to(cuda)
    plain.mhc.load_state_dict(drops.mhc.state_dict())
    res, br, w = torch.randn(30, 128, device=cuda), torch.randn(30, 128, device=cuda), torch.ones(128, device=cuda)
    groups = mhc.dropout_groups(br.shape)
    for turn in range(2):
        a, b = br.clone().requires_grad_(True), br.clone().requires_grad_(True)
        out = drops(res, a)
        want = plain(res, mhc.dropout(b, 0.25, (11, 2 * turn * groups)))
        assert torch.equal(out, want)
        out.square().sum().backward()
        want.square().sum().backward()
        assert torch.equal(a.grad, b.grad)
        for x, y in zip(drops.forward_prenorm(res, br, w),
                        plain.forward_prenorm(res, mhc.dropout(br, 0.25, (11, (2 * turn + 1) * groups)), w)):
            assert torch.equal(x, y)
    drops.eval(), plain.eval()
    with torch.no_grad():
        assert torch.equal(drops(res, br), plain(res, br))
    again = mhc.MHCResidualWrapper(128, n, branch_dropout=0.25, **kw)
    again.load_state_dict(drops.state_dict())
    assert again.branch_dropout.counter.state.tolist() == [11, 4 * groups]


def test_example_with_dropout_answers(cuda):
    spec = importlib.util.spec_from_file_location("train_streams", os.path.join(ROOT, "examples", "train_streams.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    losses, kept, ids, logprobs = m.train(steps=2, batch=2, length=16, vocab=50, dropout=0.1, answer=True)
    again = m.train(steps=2, batch=2, length=16, vocab=50, dropout=0.1)[0]
    assert losses[0] == again[0]  # the masks are the seed's
    assert ids.shape == (16, 5) and bool((logprobs[:, :-1] >= logprobs[:, 1:]).all())
    logits = torch.randn(20, 50, device=cuda, requires_grad=True)
    targets = torch.randint(0, 50, (20,), device=cuda)
    targets[:4] = 0
    (g,) = torch.autograd.grad(m.loss_of(logits, targets), logits)
    x = logits.detach().double().requires_grad_(True)
    want = torch.nn.functional.cross_entropy(x, targets, ignore_index=0)
    (e,) = torch.autograd.grad(want, x)
    assert (g.double() - e).abs().max() < 64 * U * e.abs().max()
