"""The distillation loss where a teacher's list repeats words: tau^2 KL(p || q) with p over the words, a word's
probability the sum of its entries'.

The bounds are those of the head's own tests, and for a word of r entries a sum of r probabilities (each off by at most
2^-20 of itself: an exponential and a sum over the list) in fp32: r 2^-24 more of P in P log P, whose derivative is
1 + log P."""
import math

import pytest
import torch

import test_gpu_lm_ends
from pragnosia_amd.head import linear_distill
from test_gpu_head import inputs, near, oracle as by_entry

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def oracle(h, W, y=None, g_ce=None, g_lse=None, ids=None, z=None, tau=1.0, g_kd=None):
    """The head's oracle, with the distillation loss of the words' probabilities."""
    out = by_entry(h, W, y, g_ce, g_lse, ids, z, tau, g_kd)
    if ids is None:
        return out
    V = W.shape[0]
    x = h.detach().bfloat16().double() @ W.detach().bfloat16().double().t()
    on = (ids >= 0) & (ids < V)
    zt = (z.double() / tau).masked_fill(~on, -math.inf)
    some = zt.amax(1) > -math.inf
    p = torch.where(some[:, None], torch.softmax(zt.masked_fill(~some[:, None], 0), 1), 0) * on
    at = ids.clamp(0, V - 1)
    P = torch.zeros_like(x).scatter_add_(1, at, p)
    repeats = torch.zeros_like(x).scatter_add_(1, at, on.double())
    kd = tau * tau * (torch.xlogy(P, P) - P * torch.log_softmax(x / tau, 1)).sum(1)
    added = (P * (1 + torch.where(P > 0, P.log().abs(), 0)) * (repeats * U + 2.0 ** -20)).sum(1)
    out["kd"] = kd, out["kd"][1] + tau * tau * added
    return out


@pytest.mark.parametrize("K", [2, 4, 65, 1000])
def test_one_word(K):
    """A list of one word over and over is certain of it: the loss is -tau^2 log q of that word, however long the
    list."""
    n, V, d = 9, 50, 64
    h, W, _, g = inputs(n, V, d, seed=K)
    word = torch.randint(0, V, (n, 1), generator=g).cuda()
    z = torch.randn(n, K, generator=g).cuda()
    for tau in (1.0, 2.0):
        kd, _ = linear_distill(h, W, word.expand(n, K), z, tau)
        x = h.double() @ W.double().t()
        want = -tau * tau * torch.log_softmax(x / tau, 1).gather(1, word)[:, 0]
        near(kd, (want, oracle(h, W, ids=word.expand(n, K), z=z, tau=tau)["kd"][1]), "kd")
        assert (kd > 0).all()


def test_two_entries_of_four_words():
    """Student logits 3, 0, 0, 0 and the first word twice: log(e^3 + 3) - 3 = 0.1391."""
    h = torch.tensor([[3.0] + 7 * [0.0]], device="cuda").bfloat16()
    W = torch.eye(4, 8, device="cuda").bfloat16()
    kd, _ = linear_distill(h, W, torch.zeros(1, 2, dtype=torch.long, device="cuda"), torch.ones(1, 2, device="cuda"))
    assert abs(kd.item() - (math.log(math.exp(3) + 3) - 3)) <= 2.0 ** -19


@pytest.mark.parametrize("n,V,d,K,tau", [(40, 12, 64, 5, 1.0), (70, 30, 72, 64, 2.0), (33, 300, 136, 200, 0.5),
                                         (20, 90, 64, 1000, 3.0)])
@pytest.mark.parametrize("labels", [False, True])
def test_some_words_repeated(n, V, d, K, tau, labels):
    """Lists drawn with replacement, some entries absent, without probability or of the type's lowest value."""
    h, W, y, g = inputs(n, V, d, seed=K)
    y = y if labels else None
    ids, z = torch.randint(-1, V + 1, (n, K), generator=g).cuda(), 3 * torch.randn(n, K, generator=g).cuda()
    z[torch.rand(n, K, generator=g).cuda() < 0.1] = -math.inf
    z[1] = -math.inf
    z[2], ids[2] = torch.finfo(torch.float32).min, ids[2, 0].clamp(0, V - 1)
    plain = z.clone()
    plain[2] = 0
    g_kd, g_ce = torch.randn(n, generator=g).cuda(), torch.randn(n, generator=g).cuda()
    want = oracle(h, W, y, None, None, ids, plain, tau)["kd"][0]
    # the bounds and gradients with -60 for -inf (a relative 2^-28 of a probability at tau = 3), as they take the
    # logits' size; row 1, where nothing is left, has no gradient
    finite = oracle(h, W, y, g_ce if labels else None, None, ids, plain.masked_fill(plain == -math.inf, -60.0), tau,
                    torch.where(torch.arange(n, device="cuda") == 1, 0, g_kd))
    a, b = h.clone().requires_grad_(), W.clone().requires_grad_()
    kd, ce = linear_distill(a, b, ids, z, tau, y)
    near(kd, (want, finite["kd"][1]), "kd")
    assert kd[1] == 0 and (kd >= -finite["kd"][1]).all()
    dh, dW = torch.autograd.grad((kd, ce) if labels else kd, (a, b), (g_kd, g_ce) if labels else g_kd)
    near(dh, finite["dh"], "dh", 2.0 ** -8), near(dW, finite["dW"], "dW", 2.0 ** -8)


def test_rows_without_repeats_keep_their_bits():
    """A row's loss is its own: the same bits beside rows that repeat words and by itself."""
    n, V, d, K = 16, 200, 64, 70
    h, W, _, g = inputs(n, V, d, seed=3)
    ids = torch.stack([torch.randperm(V, generator=g)[:K] for _ in range(n)]).cuda()
    z = torch.randn(n, K, generator=g).cuda()
    want, _ = linear_distill(h, W, ids, z, 2.0)
    mixed = ids.clone()
    mixed[::2, 1:9] = mixed[::2, :1]
    got, _ = linear_distill(h, W, mixed, z, 2.0)
    assert torch.equal(got[1::2], want[1::2]) and (got[::2] != want[::2]).all()


@pytest.mark.parametrize("mixer", ["aspin", "dspin"])
def test_training_step(monkeypatch, mixer):
    """The model's whole step with a teacher that repeats words, its losses against this oracle."""
    monkeypatch.setattr(test_gpu_lm_ends, "oracle", oracle)
    test_gpu_lm_ends.test_training_step(mixer, True)
