"""Every tile of the head's kernels against the formulas in 64 bits (the bounds of the head's own tests), and rows past
2^31 elements on inputs whose bounds are far below the results.

The tile of the forward's logits is read off its workspace, whose size counts two pieces a tile of words. The rule for
the backward's tiles and cuts gives, for these sizes: logits' gradients in 256 x 256, 192 x 256, 128 x 128 and 64 x 64;
the products in 256 x 256, 192 x 256 and 128 x 128, whole and cut along words, along tokens, and by pieces."""
import pytest
import torch

from pragnosia_amd.head import _workspace, linear_cross_entropy, linear_distill
from test_gpu_head import inputs, near, oracle

pytestmark = pytest.mark.gpu


def words_of_tile(n, V, d, K):
    """Words of the forward's tile, by the pieces that its workspace has room for (None if two tiles give the same)."""
    pieces = (_workspace("pragnosia_head_fwd_workspace_bytes", n, V, d, K) // (4 * n) - 2) // 3
    fits = [x for x in (256, 192, 128, 64) if 2 * -(-V // x) == pieces]
    return fits[0] if len(fits) == 1 else None


def teacher_of(n, V, K, g):
    """K different words a token, lists cut short at random, on the GPU (permutations take the host too long)."""
    gd = torch.Generator(device="cuda").manual_seed(int(torch.randint(1 << 30, (1,), generator=g)))
    ids = torch.rand(n, V, generator=gd, device="cuda").topk(K, 1).indices
    keep = torch.randint(0, K + 1, (n, 1), generator=gd, device="cuda")
    return torch.where(torch.arange(K, device="cuda") < keep, ids, -1), 3 * torch.randn(n, K, generator=gd,
                                                                                       device="cuda")


#  tokens, words, width: forward's tile
@pytest.mark.parametrize("n,V,d,tile", [
    (7, 8192, 768, 64),       # products 128 x 128, dh cut along the words
    (1001, 10007, 512, 192),  # dl 192 x 256; products 192 x 256, dh cut along the words
    (2049, 8190, 704, 192),   # products 128 x 128
    (6000, 3001, 768, 192),   # products 192 x 256, dW cut along the tokens
    (4001, 4099, 1000, 192),  # products 192 x 256, whole
    (8190, 8192, 704, 256),   # dl 256 x 256; products 192 x 256
    (4096, 8192, 1024, 256),  # products 256 x 256, dh cut
    (9001, 20011, 768, 256),  # pieces of the vocabulary in large tiles
])
def test_cross_entropy(n, V, d, tile):
    assert words_of_tile(n, V, d, 0) == tile
    h, W, y, g = inputs(n, V, d, seed=n)
    g_ce, g_lse = torch.rand(n, generator=g).cuda() / n, torch.randn(n, generator=g).cuda() / (8 * n)
    h.requires_grad_(), W.requires_grad_()
    loss, lse = linear_cross_entropy(h, W, y)
    dh, dW = torch.autograd.grad((loss, lse), (h, W), (g_ce, g_lse))
    want = oracle(h, W, y, g_ce, g_lse)
    near(loss, want["ce"], "ce"), near(lse, want["lse"], "lse")
    near(dh, want["dh"], "dh", 2.0 ** -8), near(dW, want["dW"], "dW", 2.0 ** -8)


@pytest.mark.parametrize("n,V,d,K,tau,labels,tile", [
    (200, 8192, 768, 16, 1.0, True, 64),
    (1500, 12001, 704, 100, 1.0, False, 192),  # products 256 x 256
    (2049, 8190, 704, 20, 2.0, True, 192),     # two exponentials
    (1999, 30011, 768, 33, 2.0, True, 256),    # two exponentials; products 256 x 256
    (4096, 8192, 1024, 1000, 1.0, True, 256),  # the longest rows of W held in registers; a long list
    (300, 2000, 1032, 1024, 0.5, True, 64),    # past them; the longest list
    (8190, 8192, 512, 128, 4.0, False, 256),
    (9001, 20011, 768, 32, 1.5, True, 256),    # pieces of the vocabulary in large tiles
])
def test_distill(n, V, d, K, tau, labels, tile):
    assert words_of_tile(n, V, d, K) == tile
    h, W, y, g = inputs(n, V, d, seed=n)
    ids, z = teacher_of(n, V, K, g)
    y = y if labels else None
    g_kd, g_ce = torch.rand(n, generator=g).cuda() / n, torch.rand(n, generator=g).cuda() / n
    h.requires_grad_(), W.requires_grad_()
    kd, ce = linear_distill(h, W, ids, z, tau, y)
    grads = torch.autograd.grad((kd, ce) if labels else kd, (h, W), (g_kd, g_ce) if labels else g_kd)
    want = oracle(h, W, y, g_ce if labels else None, None, ids, z, tau, g_kd)
    near(kd, want["kd"], "kd")
    if labels:
        near(ce, want["ce"], "ce")
    near(grads[0], want["dh"], "dh", 2.0 ** -8), near(grads[1], want["dW"], "dW", 2.0 ** -8)


@pytest.mark.parametrize("n,V", [(3, 33000), (33000, 24)])
def test_rows_past_32_bits(n, V):
    """A table, and hidden rows, of more than 2^31 elements, with sixteen values of +-1 in each of the long operand's
    rows (its last column among them) and of +-1/16 all over the other's: a logit sums sixteen products of 1/16, so its
    bound is small beside every gradient, and results of zeros, or of other rows, are off."""
    d, g = 65536, torch.Generator(device="cuda").manual_seed(21)
    sign = lambda *s: (torch.randint(0, 2, s, generator=g, device="cuda") * 2 - 1).bfloat16()
    rows = max(n, V)
    cols = torch.randint(0, d, (rows, 16), generator=g, device="cuda")
    cols[:, -1] = d - 1
    long = torch.zeros(rows, d, device="cuda", dtype=torch.bfloat16).scatter_(1, cols, sign(rows, 16))
    short = 0.0625 * sign(min(n, V), d)
    h, W = (short, long) if n < V else (long, short)
    assert long.numel() > 2 ** 31
    h.requires_grad_(), W.requires_grad_()
    ids = torch.full((n, 4), -1, device="cuda")
    ids[:, 0], ids[-1] = torch.randint(0, V, (n,), generator=g, device="cuda"), torch.arange(V - 4, V, device="cuda")
    z = torch.randn(n, 4, generator=g, device="cuda")
    y = torch.randint(0, V, (n,), generator=g, device="cuda")
    y[0], y[-1] = 0, V - 1
    g_kd, g_ce = (0.5 + torch.rand(n, generator=g, device="cuda") for _ in range(2))
    kd, ce = linear_distill(h, W, ids, z, 2.0, y)
    dh, dW = torch.autograd.grad((kd, ce), (h, W), (g_kd, g_ce))
    want = oracle(h, W, y, g_ce, None, ids, z, 2.0, g_kd)
    near(kd, want["kd"], "kd"), near(ce, want["ce"], "ce")
    assert (want["kd"][1] < 0.1).all() and (want["ce"][1] < 0.1).all()
    past = 2 ** 31 // d  # the first row that starts there
    for got, name in ((dh, "dh"), (dW, "dW")):
        ref, err = want.pop(name)
        near(got, (ref, err), name, 2.0 ** -8)
        # the bound would not pass zeros or the negative: it is a quarter of the gradient at most. (The short operand's
        # last column sums all the long one's rows, of either sign: its bound is no smaller than it.)
        for part in ([slice(None), slice(past, None), slice(-1, None)] if ref.shape[0] == rows else [slice(None)]):
            r, e = (ref, err) if ref.shape[0] == rows else (ref[:, :-1], err[:, :-1])
            assert (e[part].norm() < 0.25 * r[part].norm()) and r[part].any()


def test_longest_batch():
    """2^24 tokens, the most there may be. Positive hidden rows and one label, so that no sum cancels: an fp32 sum over
    the tokens, 32 products a step, is off by (2^24 / 32 + 64) 2^-24 of itself at most, 3.2%."""
    n, V, d = 1 << 24, 24, 8
    g = torch.Generator(device="cuda").manual_seed(31)
    h = (0.5 + torch.rand(n, d, generator=g, device="cuda")).bfloat16().requires_grad_()
    W = torch.randn(V, d, generator=g, device="cuda").bfloat16().requires_grad_()
    y = torch.where(torch.rand(n, generator=g, device="cuda") < 0.1, -100, 3)
    y[0], y[-1] = 3, 3
    loss, lse = linear_cross_entropy(h, W, y)
    dh, dW = torch.autograd.grad(loss.sum(), (h, W))
    want_dW = torch.zeros(V, d, device="cuda", dtype=torch.float64)
    with torch.no_grad():
        for a in range(0, n, 1 << 21):
            part = slice(a, a + (1 << 21))
            want = oracle(h[part], W, y[part], torch.ones(1 << 21, device="cuda"))
            near(loss[part], want["ce"], "ce"), near(lse[part], want["lse"], "lse")
            near(dh[part], want["dh"], "dh", 2.0 ** -8)
            want_dW += want["dW"][0]
    # (dl's rounding and the logits' errors, 2^-7 of it in all, and the result's rounding)
    assert ((dW.double() - want_dW).abs() <= (0.032 + 2.0 ** -7 + 2.0 ** -8) * want_dW.abs()).all()


def test_largest_vocabulary():
    """2^24 words. A row's 2^19 pieces of 32 words (eight a lane, two exchanges) are joined by 64 threads, 8192 one by
    one, and six steps: the sum of exponentials is off by 8300 2^-24 of itself at most, 2^-10.9."""
    n, V, d = 5, 1 << 24, 8
    g = torch.Generator(device="cuda").manual_seed(32)
    h = torch.randn(n, d, generator=g, device="cuda").bfloat16().requires_grad_()
    W = torch.randn(V, d, generator=g, device="cuda").bfloat16().requires_grad_()
    y = torch.tensor([0, V - 1, V, V // 2 + 1, 12345], device="cuda")
    loss, lse = linear_cross_entropy(h, W, y)
    dh, dW = torch.autograd.grad(loss.sum(), (h, W))
    with torch.no_grad():
        h64, W64 = h.double(), W.double()
        x = h64 @ W64.t()
        want = torch.logsumexp(x, 1)
        assert ((lse - want).abs() <= 2.0 ** -10.9).all()
        on = y < V
        label = x.gather(1, y.clamp(max=V - 1)[:, None])[:, 0]
        assert ((loss - torch.where(on, want - label, 0)).abs() <= 2.0 ** -10.9).all()
        dl = (x - want[:, None]).exp()
        dl[torch.arange(n), y.clamp(max=V - 1)] -= 1
        dl *= on[:, None]
        # an element of dl: 2^-10.9 for the sum, 2^-8 for its rounding, 2^-7.8 in all; dh sums 57 pieces of the words,
        # in parts of at most 2^13, 32 a step: 1100 2^-24 of the magnitudes at most
        full = dl.abs() @ W64.abs()
        assert ((dh - dl @ W64).abs() <= (2.0 ** -7.8 + 2.0 ** -13) * full + 2.0 ** -8 * (dl @ W64).abs()).all()
        want, full = dl.t() @ h64, dl.abs().t() @ h64.abs()
        assert ((dW - want).abs() <= (2.0 ** -7.8 + 2.0 ** -20) * full + 2.0 ** -8 * want.abs()).all()
        assert dW[y[on]].abs().amax(1).min() > 0.1 and dW[-2].any()
