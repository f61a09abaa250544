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


def ce_grads(h, W, y, g):
    h, W = h.detach().requires_grad_(), W.detach().requires_grad_()
    loss, lse = linear_cross_entropy(h, W, y)
    return [loss.detach(), lse.detach(), *torch.autograd.grad(loss, (h, W), g)]


def test_one_gradient_at_a_time():
    """dh or dW alone, and the gradient of one output alone, are those of the whole call."""
    h, W, y, g = inputs(100, 300, 72, seed=3)
    gc = torch.randn(100, generator=g).cuda()
    both = ce_grads(h, W, y, gc)
    a = h.clone().requires_grad_()
    assert torch.equal(torch.autograd.grad(linear_cross_entropy(a, W, y)[0], a, gc)[0], both[2])
    b = W.clone().requires_grad_()
    assert torch.equal(torch.autograd.grad(linear_cross_entropy(h, b, y)[0], b, gc)[0], both[3])
    lse, = torch.autograd.grad(linear_cross_entropy(a, W, y)[1], a, gc)
    near(lse, oracle(h, W, y, None, gc)["dh"], "dh of lse", 2.0 ** -8)
    with torch.no_grad():
        assert torch.equal(linear_cross_entropy(h, W, y)[0], both[0])


def test_fp32_operands():
    """fp32 h and W are rounded to bf16 for the products; dh comes in fp32, and dW in fp32 without a last rounding."""
    h, W, y, g = inputs(130, 260, 64, seed=4, dtype=torch.float32)
    gc = torch.randn(130, generator=g).cuda()
    want = oracle(h, W, y, gc)
    loss, lse, dh, dW = ce_grads(h, W, y, gc)
    assert dh.dtype == dW.dtype == torch.float32
    near(loss, want["ce"], "ce"), near(dh, want["dh"], "dh", 2.0 ** -8), near(dW, want["dW"], "dW", 2.0 ** -23)


def test_leading_shapes_strides_and_offsets():
    """(B, T, d) hidden rows cut out of longer sequences, a table inside a larger buffer at an odd offset, int32 labels,
    a transposed list of entries: the same bits as the dense call."""
    g = torch.Generator().manual_seed(5)
    full = torch.randn(3, 21, 64, generator=g).bfloat16().cuda()
    h = full[:, :-1]
    buf = torch.randn(200 * 64 + 3, generator=g).bfloat16().cuda()
    W = buf[3:].view(200, 64)
    assert not h.is_contiguous() and W.data_ptr() % 16
    y = torch.randint(0, 200, (3, 21), generator=g).cuda()[:, 1:]
    gc = torch.randn(3, 20, generator=g).cuda()
    got = ce_grads(h, W, y.int(), gc)
    want = ce_grads(h.reshape(60, 64).clone(), W.clone(), y.reshape(60).clone(), gc.reshape(60))
    assert got[0].shape == (3, 20) and got[2].shape == h.shape
    assert all(torch.equal(a.reshape(b.shape), b) for a, b in zip(got, want))
    ids, z = torch.randint(-1, 200, (5, 60), generator=g).cuda().t(), torch.randn(5, 60, generator=g).cuda().t()
    kd, _ = linear_distill(h, W, ids.reshape(3, 20, 5), z.double().reshape(3, 20, 5), 1.5)
    dense, _ = linear_distill(h.reshape(60, 64), W, ids.contiguous(), z.contiguous(), 1.5)
    assert torch.equal(kd.reshape(60), dense)


def test_nothing_to_do():
    h, W, y, _ = inputs(0, 50, 64)
    loss, lse, dh, dW = ce_grads(h, W, y, torch.zeros(0, device="cuda"))
    assert loss.shape == lse.shape == (0,) and dh.shape == (0, 64) and not dW.any() and dW.shape == W.shape
    h, W, y, _ = inputs(40, 50, 64, pad=1.1)  # every label padding
    loss, lse, dh, dW = ce_grads(h, W, y, torch.ones(40, device="cuda"))
    assert not loss.any() and not dh.any() and not dW.any() and torch.isfinite(lse).all()
    loss, _, dh, dW = ce_grads(*inputs(40, 50, 64)[:3], torch.zeros(40, device="cuda"))  # weights of zero
    assert loss.any() and not dh.any() and not dW.any()


def test_masked_rows_hold_nothing():
    """A padded row's NaN or infinity stays in its own lse: other rows' losses, and (with finite rows there) the
    gradients, are those without it; weights of any size on padded labels change nothing."""
    h, W, y, g = inputs(300, 270, 64, seed=6)
    gc = torch.rand(300, generator=g).cuda()
    y[::7] = -100
    want = ce_grads(h, W, y, gc)
    big = torch.where(y < 0, 1e30, gc)
    assert all(((a.double() - b.double()).norm() <= 2.0 ** -7 * b.double().norm())
               for a, b in zip(ce_grads(h, W, y, big), want))
    bad = h.clone()
    bad[0], bad[7] = float("nan"), float("inf")
    loss, lse = linear_cross_entropy(bad, W, y)
    keep = torch.ones(300, dtype=torch.bool, device="cuda")
    keep[0] = keep[7] = False
    assert torch.equal(loss, want[0]) and torch.equal(lse[keep], want[1][keep]) and not torch.isfinite(lse[~keep]).any()
    dh, = torch.autograd.grad(linear_cross_entropy(bad.requires_grad_(), W, y)[0], bad, gc)
    assert torch.equal(dh, want[2])  # zero rows there


def test_teacher_edges():
    """Entries that are not there hold anything; -inf has no probability; the type's lowest value in a whole row is a
    uniform one; a repeated id is one entry of the summed probability; a label among the entries."""
    n, V, d = 6, 90, 64
    h, W, y, g = inputs(n, V, d, seed=7, pad=0)
    ids = torch.stack([torch.randperm(V, generator=g)[:5] for _ in range(n)]).cuda()
    z = torch.randn(n, 5, generator=g).cuda()
    inf, nan, low = float("inf"), float("nan"), torch.finfo(torch.float32).min
    ids[0, 2], z[0, 2] = -1, nan
    ids[1, 0], z[1, 0] = V, inf
    z[2, 1] = -inf
    z[3] = -inf
    z[4] = low
    ids[5] = ids[5, 0]
    ids[2, 3] = y[2]
    plain_z = z.clone()
    plain_z[0, 2], plain_z[1, 0], plain_z[4] = 0, 0, 0
    g_kd, g_ce = torch.randn(n, generator=g).cuda(), torch.randn(n, generator=g).cuda()
    for tau in (1.0, 0.25, 3.0):
        # the oracle sums a repeated id's entropy by entry, as the definition does
        want = oracle(h, W, y, g_ce, None, ids, plain_z.masked_fill(plain_z == -inf, -1e9), tau, g_kd)
        a, b = h.clone().requires_grad_(), W.clone().requires_grad_()
        kd, ce = linear_distill(a, b, ids, z, tau, y)
        live = torch.tensor([0, 1, 2, 4, 5], device="cuda")
        assert kd[3] == 0
        near(kd[live], tuple(t[live] for t in want["kd"]), "kd"), near(ce, want["ce"], "ce")
        dh, dW = torch.autograd.grad((kd, ce), (a, b), (g_kd, g_ce))
        w3 = g_kd.clone()
        w3[3] = 0
        want = oracle(h, W, y, g_ce, None, ids, plain_z.masked_fill(plain_z == -inf, -1e9), tau, w3)
        near(dh, want["dh"], "dh", 2.0 ** -8), near(dW, want["dW"], "dW", 2.0 ** -8)


def test_teacher_that_is_no_distribution():
    """A NaN or +inf among a token's present logits (and a whole row of NaN) is a NaN loss of that token; the others
    keep their bits, the cross entropy too."""
    n, V, d = 7, 90, 64
    h, W, y, g = inputs(n, V, d, seed=17, pad=0)
    ids = torch.stack([torch.randperm(V, generator=g)[:70] for _ in range(n)]).cuda()
    z = torch.randn(n, 70, generator=g).cuda()
    want = linear_distill(h, W, ids, z, 2.0, y)
    bad = z.clone()
    bad[1, 3], bad[2, 69], bad[4], bad[5, 0] = float("nan"), float("nan"), float("nan"), float("inf")
    kd, ce = linear_distill(h, W, ids, bad, 2.0, y)
    assert kd[[1, 2, 4, 5]].isnan().all()
    assert torch.equal(kd[[0, 3, 6]], want[0][[0, 3, 6]]) and torch.equal(ce, want[1])


def test_gradient_against_differences():
    """The directional derivative of the summed losses, by central differences of the formula in 64 bits, along random
    directions: the kernel's gradient gives it to its bf16 rounding (2^-7 of the norms of gradient and direction)."""
    n, V, d = 20, 70, 64
    h, W, y, g = inputs(n, V, d, seed=8)
    ids, z = teacher(n, V, 6, g)
    h.requires_grad_(), W.requires_grad_()
    kd, ce = linear_distill(h, W, ids, z, 2.0, y)
    grads = torch.autograd.grad(kd.sum() + 0.5 * ce.sum(), (h, W))

    def f(hh, ww):
        x = hh @ ww.t()
        on = ids >= 0
        some = on.any(1)
        p = torch.softmax((z.double() / 2).masked_fill(~on, -math.inf)[some], 1)
        lq = torch.log_softmax(x / 2, 1).gather(1, ids.clamp(min=0))[some]
        k = 4 * (torch.xlogy(p, p) - p * lq).sum()
        v = y >= 0
        return k + 0.5 * F.cross_entropy(x[v], y[v], reduction="sum")

    h64, W64 = h.detach().double(), W.detach().double()
    for seed in range(3):
        gg = torch.Generator().manual_seed(seed)
        dh, dW = torch.randn(n, d, generator=gg).double().cuda(), torch.randn(V, d, generator=gg).double().cuda()
        e = 1e-5
        diff = (f(h64 + e * dh, W64 + e * dW) - f(h64 - e * dh, W64 - e * dW)) / (2 * e)
        got = (grads[0].double() * dh).sum() + (grads[1].double() * dW).sum()
        size = grads[0].double().norm() * dh.norm() + grads[1].double().norm() * dW.norm()
        assert abs(got - diff) <= 2.0 ** -7 * size


def test_streams_and_repeated_calls():
    """Two calls at once on streams of their own, and the same call again: the same bits as one after the other."""
    a, b = inputs(700, 900, 136, seed=9), inputs(90, 5000, 64, seed=10)
    ga, gb = torch.rand(700, device="cuda"), torch.rand(90, device="cuda")
    want = ce_grads(*a[:3], ga), ce_grads(*b[:3], gb)
    torch.cuda.synchronize()
    s, t = torch.cuda.Stream(), torch.cuda.Stream()
    got = []
    for _ in range(3):
        with torch.cuda.stream(s):
            x = ce_grads(*a[:3], ga)
        with torch.cuda.stream(t):
            y = ce_grads(*b[:3], gb)
        got.append((x, y))
    torch.cuda.synchronize()
    for pair in got:
        for u, v in zip(pair, want):
            assert all(torch.equal(p, q) for p, q in zip(u, v))


def test_captured_and_replayed():
    """Forward and backward in one graph: replays on new inputs, with eager calls and synchronizations between them."""
    h, W, y, g = inputs(200, 600, 72, seed=11)
    gc = torch.rand(200, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ce_grads(h, W, y, gc)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ce_grads(h, W, y, gc)
    for seed in range(3):
        h2, W2, y2, _ = inputs(200, 600, 72, seed=20 + seed)
        h.copy_(h2), W.copy_(W2), y.copy_(y2)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(out, ce_grads(h2, W2, y2, gc)))


def test_twice_differentiated_is_refused():
    h, W, y, _ = inputs(10, 20, 64)
    h.requires_grad_()
    dh, = torch.autograd.grad(linear_cross_entropy(h, W, y)[0].sum(), h, create_graph=True)
    with pytest.raises(RuntimeError):
        dh.sum().backward()


# every tile of the logits and of the products, cut into ranges and not
@pytest.mark.parametrize("n,V,d", [(1, 9000, 768), (129, 8192, 256), (1300, 1030, 264), (2100, 2050, 200),
                                   (4096, 520, 512), (1000, 3001, 1032)])
def test_tiles(n, V, d):
    h, W, y, g = inputs(n, V, d, seed=12)
    gc = torch.full((n,), 1.0 / n, device="cuda")
    want = oracle(h, W, y, gc)
    loss, lse, dh, dW = ce_grads(h, W, y, gc)
    near(loss, want["ce"], "ce"), near(lse, want["lse"], "lse")
    near(dh, want["dh"], "dh", 2.0 ** -8), near(dW, want["dW"], "dW", 2.0 ** -8)


@pytest.mark.parametrize("n,V", [(3, 33000), (33000, 24)])
def test_offsets_past_32_bits(n, V):
    """A table, and hidden rows, of more than 2^31 elements: losses and gradients up to the last row."""
    d, g = 65536, torch.Generator(device="cuda").manual_seed(11)
    h = torch.randn(n, d, generator=g, device="cuda", dtype=torch.bfloat16).requires_grad_()
    W = torch.randn(V, d, generator=g, device="cuda", dtype=torch.bfloat16).mul_(2 * d ** -0.5).requires_grad_()
    assert max(h.numel(), W.numel()) > 2 ** 31
    ids = torch.randint(0, V, (n, 4), generator=g, device="cuda").sort(1).values
    ids[:, 1:] = torch.where(ids[:, 1:] == ids[:, :-1], -1, ids[:, 1:])
    ids[-1], z = torch.arange(V - 4, V, device="cuda"), torch.randn(n, 4, generator=g, device="cuda")
    y = torch.randint(0, V, (n,), generator=g, device="cuda")
    y[0], y[-1] = 0, V - 1
    g_kd, g_ce = torch.randn(n, generator=g, device="cuda"), torch.randn(n, generator=g, device="cuda")
    kd, ce = linear_distill(h, W, ids, z, 2.0, y)
    dh, dW = torch.autograd.grad((kd, ce), (h, W), (g_kd, g_ce))
    want = oracle(h, W, y, g_ce, None, ids, z, 2.0, g_kd)
    near(kd, want["kd"], "kd"), near(ce, want["ce"], "ce")
    near(dh, want.pop("dh"), "dh", 2.0 ** -8), near(dW, want.pop("dW"), "dW", 2.0 ** -8)
