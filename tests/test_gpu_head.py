"""The head's losses (cross entropy, distillation) and their gradients against the formulas in 64 bits.

Tolerances, from the operations: a logit is d products of bf16 values summed in fp32 (off by at most (d + 2) 2^-24
sum |h w|); an exponential's argument is rounded to 2^-23 of its size and the hardware exponential to about 2^-22; a
softmax sum over V terms adds V 2^-24 at most. A logit's gradient is rounded to bf16 once (2^-8 of it), the products'
sums are fp32 and the results rounded to bf16 (2^-8)."""
import math

import pytest
import torch
import torch.nn.functional as F

from pragnosia_amd.head import linear_cross_entropy, linear_distill

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def inputs(n, V, d, seed=0, spread=2.0, pad=0.1, dtype=torch.bfloat16):
    g = torch.Generator().manual_seed(seed)
    h = F.layer_norm(torch.randn(n, d, generator=g), (d,)).to(dtype).cuda()
    W = (spread * d ** -0.5 * torch.randn(V, d, generator=g)).to(dtype).cuda()
    y = torch.randint(0, V, (n,), generator=g)
    y[torch.rand(n, generator=g) < pad] = -100
    return h, W, y.cuda(), g


def teacher(n, V, K, g, short=True):
    ids = torch.stack([torch.randperm(max(V, K), generator=g)[:K] for _ in range(n)])  # some past V where K > V
    z = 3 * torch.randn(n, K, generator=g)
    if short:
        keep = torch.randint(0, K + 1, (n, 1), generator=g)
        ids[torch.arange(K) >= keep] = -1
    return ids.cuda(), z.cuda()


def oracle(h, W, y=None, g_ce=None, g_lse=None, ids=None, z=None, tau=1.0, g_kd=None):
    """Values, gradients and the bounds of their errors, by the definitions in 64 bits."""
    h, W = h.detach().bfloat16().double(), W.detach().bfloat16().double()
    V, d = W.shape
    x = h @ W.t()
    dx_l = (d + 2) * U * (h.abs() @ W.abs().t()) + 2.0 ** -22 * (x.abs() + 1)  # of a logit, and of an exponent
    lse = torch.logsumexp(x, 1)
    e_lse = dx_l.amax(1) + (V + 32) * U + 2.0 ** -22 * (1 + lse.abs())
    out, dl, size, rel = {}, torch.zeros_like(x), torch.zeros_like(x), 0.0
    if y is not None:
        on = (y >= 0) & (y < V)
        at = y.clamp(0, V - 1)
        label = x.gather(1, at[:, None])[:, 0]
        out["lse"], out["ce"] = (lse, e_lse), (torch.where(on, lse - label, 0), 2 * e_lse + 2.0 ** -22 * label.abs())
        gc = torch.zeros_like(lse) if g_ce is None else torch.where(on, g_ce.double(), 0)
        gs = torch.zeros_like(lse) if g_lse is None else g_lse.double()
        p = (x - lse[:, None]).exp()
        hot = F.one_hot(at, V)
        dl += (gc + gs)[:, None] * p - gc[:, None] * hot
        size += (gc.abs() + gs.abs())[:, None] * p + gc.abs()[:, None] * hot
        rel = 2 * (dx_l + e_lse[:, None]) + 2.0 ** -20
    if ids is not None:
        on = (ids >= 0) & (ids < V)
        zt = (z.double() / tau).masked_fill(~on, -math.inf)
        some = zt.amax(1) > -math.inf
        pt = torch.where(some[:, None], torch.softmax(zt.masked_fill(~some[:, None], 0), 1), 0) * on
        t = torch.zeros_like(x).scatter_add_(1, ids.clamp(0, V - 1), pt)
        lq = torch.log_softmax(x / tau, 1)
        per_entry = torch.xlogy(pt, pt) - pt * lq.gather(1, ids.clamp(0, V - 1))
        out["kd"] = (tau * tau * per_entry.sum(1),
                     tau * tau * (2 * e_lse / min(tau, 1.0) + 2.0 ** -19 * (1 + x.abs().amax(1) / tau +
                                                                           torch.where(on, z.abs(), 0).amax(1) / tau)))
        if g_kd is not None:
            gk = g_kd.double()[:, None] * tau
            dl += gk * (lq.exp() * some[:, None] - t)
            size += gk.abs() * (lq.exp() * some[:, None] + t)
            rel = rel + 2 * (dx_l + e_lse[:, None]) / min(tau, 1.0) + 2.0 ** -19 * (1 + z.abs().amax() / tau)
    e_dl = dl.abs() * 2.0 ** -8 + size * rel * 1.01
    for name, a, b in (("dh", dl, W), ("dW", dl.t(), h)):
        k = a.shape[1]
        full = a.abs() @ b.abs()
        err = (e_dl if name == "dh" else e_dl.t()) @ b.abs() + k * U * full
        out[name] = (a @ b, err)
    return out


def near(got, want, what, rounded=None):
    ref, err = want
    if rounded is not None:
        err = err + rounded * (ref.abs() + err)
    off = (got.double() - ref).abs() - err
    assert torch.isfinite(got).all() and got.shape == ref.shape and (off <= 1e-30).all(), \
        (what, off.max().item(), got.double().flatten()[off.argmax()].item(), ref.flatten()[off.argmax()].item())


# one token and one word, sizes below, at and past a tile, widths that end inside a step
SHAPES = [(1, 1, 8), (1, 1000, 64), (3, 7, 72), (64, 256, 64), (257, 255, 136), (300, 1030, 704), (513, 514, 128)]


@pytest.mark.parametrize("n,V,d", SHAPES)
def test_cross_entropy(n, V, d):
    h, W, y, g = inputs(n, V, d)
    g_ce, g_lse = torch.randn(n, generator=g).cuda(), 0.1 * torch.randn(n, generator=g).cuda()
    want = oracle(h, W, y, g_ce, g_lse)
    h.requires_grad_(), W.requires_grad_()
    loss, lse = linear_cross_entropy(h, W, y)
    assert loss.dtype == lse.dtype == torch.float32 and not loss[y < 0].any()
    near(loss, want["ce"], "ce"), near(lse, want["lse"], "lse")
    dh, dW = torch.autograd.grad((loss, lse), (h, W), (g_ce, g_lse))
    assert dh.dtype == dW.dtype == torch.bfloat16
    near(dh, want["dh"], "dh", 2.0 ** -8), near(dW, want["dW"], "dW", 2.0 ** -8)


@pytest.mark.parametrize("n,V,d,K,tau", [(1, 1, 8, 1, 1.0), (1, 500, 64, 5, 2.0), (70, 300, 72, 64, 1.0),
                                         (300, 1030, 136, 33, 3.0), (130, 60, 64, 100, 0.5)])
@pytest.mark.parametrize("labels", [False, True])
def test_distill(n, V, d, K, tau, labels):
    h, W, y, g = inputs(n, V, d, seed=1)
    ids, z = teacher(n, V, K, g)
    y = y if labels else None
    g_kd, g_ce = torch.randn(n, generator=g).cuda(), torch.randn(n, generator=g).cuda()
    want = oracle(h, W, y, g_ce if labels else None, None, ids, z, tau, g_kd)
    h.requires_grad_(), W.requires_grad_()
    kd, ce = linear_distill(h, W, ids, z, tau, y)
    near(kd, want["kd"], "kd")
    assert not kd[~((ids >= 0) & (ids < V)).any(1)].any()
    if labels:
        near(ce, want["ce"], "ce")
        dh, dW = torch.autograd.grad((kd, ce), (h, W), (g_kd, g_ce))
    else:
        assert ce is None
        dh, dW = torch.autograd.grad(kd, (h, W), g_kd)
    near(dh, want["dh"], "dh", 2.0 ** -8), near(dW, want["dW"], "dW", 2.0 ** -8)


def test_several_pieces():
    """More columns than one workspace holds: dh summed over the pieces, dW piece by piece."""
    n, V, d = 2100, 60001, 64
    h, W, y, g = inputs(n, V, d, seed=2)
    ids, z = teacher(n, V, 9, g)
    g_kd, g_ce = torch.randn(n, generator=g).cuda(), torch.randn(n, generator=g).cuda()
    want = oracle(h, W, y, g_ce, None, ids, z, 2.0, g_kd)
    h.requires_grad_(), W.requires_grad_()
    kd, ce = linear_distill(h, W, ids, z, 2.0, y)
    near(kd, want["kd"], "kd"), near(ce, want["ce"], "ce")
    dh, dW = torch.autograd.grad((kd, ce), (h, W), (g_kd, g_ce))
    near(dh, want["dh"], "dh", 2.0 ** -8), near(dW, want["dW"], "dW", 2.0 ** -8)
