"""GPU: a language model's two ends together as a training step runs them -- the token lookups, the trunk, the tied
head's cross entropy and distillation losses -- piece by piece, captured in a HIP graph and traced, and each op through
torch's own checks."""
import pytest
import torch
import torch.nn.functional as F

from test_gpu_head import near, oracle
from test_gpu_training import _memset_nodes

pytestmark = pytest.mark.gpu
VOCAB, D, CTX = 1003, 128, 160


def models(mixer="aspin", seed=0):
    from pragnosia_amd.model import LM
    out = []
    for fused in (False, True):
        torch.manual_seed(seed)
        with torch.device("cuda"):
            out.append(LM(vocab=VOCAB, d=D, layers=2, mlp_mult=2, ctx=CTX, mixer=mixer, fused_ends=fused))
    with torch.no_grad():
        for m in out:
            m.e.weight.mul_(10)
    assert all(torch.equal(a, b) for a, b in zip(out[0].state_dict().values(), out[1].state_dict().values()))
    embed = out[0]._embed

    def kept(x, positions):  # the sum of the lookups, for the gradient there
        out[0]._embed_out = embed(x, positions)
        return out[0]._embed_out

    out[0]._embed = kept
    return out


def teacher(n, K, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    ids = torch.randint(0, VOCAB, (*n, K), generator=g, device="cuda")  # some twice
    ids[..., -1] = -1
    return ids, 2 * torch.randn(*n, K, generator=g, device="cuda")


def trunk(m, xs):
    with torch.autocast("cuda", dtype=torch.bfloat16):
        return m.trunk(xs[:, :-1])


def grads_of(m):
    # (a carrier may leave a parameter unused)
    return {n: p.grad.clone() for n, p in m.named_parameters() if p.grad is not None}


def clear(m):
    for p in m.parameters():
        p.grad = None


@pytest.mark.parametrize("mixer", ["aspin", "dspin"])
@pytest.mark.parametrize("kd", [False, True])
def test_training_step(mixer, kd):
    """The two ends in a step, piece by piece. The losses and their gradients of the hidden rows and the table are the
    formulas' (the bounds of the head's own tests); the whole step's gradients are, to the bit, those of the hidden
    gradient sent through the trunk, plus the head's share of the table; the trunk's are those of the model without the
    fused ends, and the lookup's share of the table is torch's to the rounding of fp32 sums (m terms: m 2^-24 of the sum
    of their magnitudes, here and there)."""
    plain, m = models(mixer)
    g = torch.Generator(device="cuda").manual_seed(1)
    xs = torch.randint(0, VOCAB, (3, CTX + 1), generator=g, device="cuda")
    y, n = xs[:, 1:], 3 * CTX
    ids, z = teacher((3, CTX), 9, 2)

    def loss_of(h):
        if not kd:
            return m.loss(h, y)
        a, b = m.distill_loss(h, ids, z, 2.0, y)
        return 0.25 * a + 0.75 * b

    # the head alone
    h = trunk(m, xs)
    leaf = h.detach().requires_grad_()
    loss = loss_of(leaf)
    dh, dW = torch.autograd.grad(loss, (leaf, m.e.weight))
    w = torch.full((n,), 1.0 / n, device="cuda")
    flat = leaf.detach().reshape(n, D)
    want = (oracle(flat, m.e.weight, y.reshape(-1), 0.75 * w, None, ids.reshape(n, -1), z.reshape(n, -1), 2.0, 0.25 * w)
            if kd else oracle(flat, m.e.weight, y.reshape(-1), w))
    parts = [(0.25, "kd"), (0.75, "ce")] if kd else [(1.0, "ce")]
    total = sum(c * want[k][0].mean() for c, k in parts)
    size = sum(c * (want[k][1].mean() + (n + 4) * 2.0 ** -24 * want[k][0].abs().mean()) for c, k in parts)
    assert abs(loss.double() - total) <= size + 2.0 ** -22 * abs(total)
    near(dh.reshape(n, D), want["dh"], "dh", 2.0 ** -8), near(dW, want["dW"], "dW", 2.0 ** -23)
    # through the trunk, and the step at once
    clear(m)
    h.backward(dh)
    pieces = grads_of(m)
    clear(m)
    loss_of(trunk(m, xs)).backward()
    whole = grads_of(m)
    for k in whole:
        assert torch.equal(whole[k], pieces[k] + dW if k == "e.weight" else pieces[k]), k
    # the model without the fused ends, from the same hidden gradient
    hp = trunk(plain, xs)
    assert torch.equal(hp, h)
    clear(plain)
    gx, = torch.autograd.grad(hp, plain._embed_out, dh, retain_graph=True)
    hp.backward(dh)
    ref = grads_of(plain)
    for k in ref:
        if k not in ("e.weight", "p.weight"):
            assert torch.equal(ref[k], pieces[k]), k
    for k, at in (("e.weight", xs[:, :-1].reshape(-1)), ("p.weight", torch.arange(CTX, device="cuda").repeat(3))):
        rows = ref[k].shape[0]
        size = torch.zeros(rows, D, device="cuda", dtype=torch.float64)
        size.index_add_(0, at, gx.reshape(n, D).double().abs())
        m_terms = torch.bincount(at, minlength=rows)[:, None]
        assert ((ref[k].double() - pieces[k].double()).abs() <= 2 * (m_terms + 2) * 2.0 ** -24 * size).all(), k


def test_captured_step():
    """The whole step (both losses) captured: no memset node; replays on new tokens, with eager steps and
    synchronizations between them, give the eager step's bits."""
    _, m = models()
    xs = torch.randint(0, VOCAB, (2, CTX + 1), device="cuda")
    ids, z = teacher((2, CTX), 5, 3)
    for p in m.parameters():
        p.grad = torch.zeros_like(p)
    out = torch.zeros((), device="cuda")

    def micro():
        with torch.autocast("cuda", dtype=torch.bfloat16):
            h = m.trunk(xs[:, :-1])
        kd, ce = m.distill_loss(h, ids, z, 1.5, xs[:, 1:])
        (kd + ce).backward()
        out.copy_((kd + ce).detach())

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            micro()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.graph(graph):
        micro()
    assert _memset_nodes(graph) == 0
    for _ in range(4):
        xs.random_(0, VOCAB)
        ids.random_(-1, VOCAB)
        got = []
        for run in (graph.replay, micro):
            for p in m.parameters():
                p.grad.zero_()
            run()
            torch.cuda.synchronize()
            got.append([out.clone()] + [p.grad.clone() for p in m.parameters()])
        for a, b in zip(*got):
            assert torch.equal(a, b)


def test_traced_step():
    """The losses and the lookup trace whole and give the eager values and gradients."""
    from pragnosia_amd.embed import embedding
    from pragnosia_amd.head import linear_cross_entropy, linear_distill
    torch._dynamo.reset()
    g = torch.Generator(device="cuda").manual_seed(4)
    W = torch.randn(VOCAB, D, generator=g, device="cuda")
    ids = torch.randint(-1, VOCAB, (2, 70), generator=g, device="cuda")
    t = teacher((2, 70), 5, 5)

    def f(W):
        h = embedding(ids, W, 0.5)
        ce, lse = linear_cross_entropy(h, W, ids)
        kd, ce2 = linear_distill(h, W, *t, 2.0, ids)
        return (ce + 0.1 * lse + kd + ce2).sum()

    grads = []
    for fn in (f, torch.compile(f, backend="aot_eager", fullgraph=True)):
        w = W.clone().requires_grad_()
        loss = fn(w)
        loss.backward()
        grads.append((loss.detach(), w.grad))
    assert (grads[0][0] - grads[1][0]).abs() <= 1e-6 * grads[0][0].abs()
    assert (grads[0][1] - grads[1][1]).norm() <= 1e-6 * grads[0][1].norm()


def test_opcheck():
    from pragnosia_amd import embed, head  # noqa: F401
    op = torch.ops.pragnosia_lm
    g = torch.Generator(device="cuda").manual_seed(6)
    h = torch.randn(20, 64, generator=g, device="cuda").bfloat16().requires_grad_()
    W = torch.randn(90, 64, generator=g, device="cuda").requires_grad_()
    y, ids = torch.randint(0, 90, (20,), device="cuda"), torch.randint(0, 90, (20, 3), device="cuda")
    z = torch.randn(20, 3, generator=g, device="cuda")
    with torch.no_grad():
        _, lse, _, stats = op.head_loss(h, W, y, ids, z, 2.0)
    gr = torch.randn(20, generator=g, device="cuda")
    samples = [("head_loss", (h, W, y, ids, z, 2.0)), ("head_loss", (h, W, y, None, None, 1.0)),
               ("head_loss", (h, W, None, ids, z, 1.0)),
               ("head_loss_bwd", (gr, None, gr, h.detach(), W.detach(), y, lse, stats, 2.0, True, True)),
               ("embed", (y, W, 2.0, False)), ("embed", (y, W, 1.0, True)),
               ("embed_bwd", (torch.randn(20, 64, generator=g, device="cuda"), y, 90, 2.0, True))]
    for name, args in samples:
        print(f"opcheck {name}", flush=True)
        torch.library.opcheck(getattr(op, name), args)


def test_lookup_is_torchs():
    """The fused model's embeddings are nn.Embedding's values; ids that torch refuses give zero rows."""
    _, m = models()
    x = torch.randint(0, VOCAB, (2, 50), device="cuda")
    assert torch.equal(m.e(x), F.embedding(x, m.e.weight))
    assert not m.e(torch.tensor([[-1, VOCAB]], device="cuda")).any()


@pytest.mark.parametrize("n", [8192, 131073])
def test_captured_losses_of_many_tokens(n):
    """The mean losses over long batches and their gradients: no memset node, every replay the eager call's bits."""
    _, m = models()
    h = torch.randn(1, n, D, device="cuda").bfloat16().requires_grad_()
    y, (ids, z) = torch.randint(0, VOCAB, (1, n), device="cuda"), teacher((1, n), 3, 6)

    def losses():
        kd, ce = m.distill_loss(h, ids, z, 1.0, y)
        loss = m.loss(h, y)
        return (kd.detach(), ce.detach(), loss.detach(), *torch.autograd.grad(kd + ce + loss, (h, m.e.weight)))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        losses()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.graph(graph):
        out = losses()
    assert _memset_nodes(graph) == 0
    for _ in range(3):
        y.random_(0, VOCAB), z.normal_()
        graph.replay()
        got = [t.clone() for t in out]
        torch.cuda.synchronize()
        for a, b in zip(got, losses()):
            assert torch.equal(a, b)
