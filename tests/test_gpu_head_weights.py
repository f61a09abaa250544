"""The head's gradients under the per-token weights that autograd hands back: weights of tokens that have no say, of
very different sizes, the same tensor for both losses, and a token taken out of one loss only."""
import math

import pytest
import torch

from pragnosia_amd.head import linear_cross_entropy, linear_distill
from test_gpu_head import ce_grads, inputs, near, oracle, teacher

pytestmark = pytest.mark.gpu
SIZES = [1e30, 3e38, math.inf, math.nan]


def kd_grads(h, W, y, ids, z, tau, g_kd, g_ce=None):
    a, b = h.detach().clone().requires_grad_(), W.detach().clone().requires_grad_()
    kd, ce = linear_distill(a, b, ids, z, tau, y)
    return torch.autograd.grad(kd if y is None else (kd, ce), (a, b), g_kd if y is None else (g_kd, g_ce))


@pytest.mark.parametrize("size", SIZES)
def test_weights_on_padded_labels(size):
    """Whatever the weight of a token without a label, the gradients keep their bits."""
    h, W, y, g = inputs(300, 270, 64, seed=6, pad=0.2)
    y[1], y[2] = 270, -1
    gc = 1e-4 * torch.rand(300, generator=g).cuda()
    there = (y >= 0) & (y < 270)
    want = ce_grads(h, W, y, torch.where(there, gc, 0))
    assert want[2].any() and want[3].any()
    for a, b in zip(ce_grads(h, W, y, torch.where(there, gc, size)), want):
        assert torch.equal(a, b)


@pytest.mark.parametrize("labels", [False, True])
@pytest.mark.parametrize("size", SIZES)
def test_weights_on_tokens_without_a_teacher(size, labels):
    """Likewise for a token whose teacher's list is empty, in the distillation loss."""
    h, W, y, g = inputs(120, 270, 64, seed=7)
    ids, z = teacher(120, 270, 6, g)
    ids[::5] = -1
    none = ~((ids >= 0) & (ids < 270)).any(1)
    gk, gc = 1e-4 * torch.rand(120, generator=g).cuda(), 1e-4 * torch.rand(120, generator=g).cuda()
    y = y if labels else None
    want = kd_grads(h, W, y, ids, z, 2.0, torch.where(none, 0, gk), gc)
    assert want[0].any() and want[1].any()
    got = kd_grads(h, W, y, ids, z, 2.0, torch.where(none, size, gk), gc)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("tau", [1.0, 3.0])
def test_one_weight_tensor_for_both_losses(tau):
    """The weights of the two losses in one tensor, or in two of equal values: the same bits."""
    h, W, y, g = inputs(300, 270, 64, seed=8)
    ids, z = teacher(300, 270, 6, g)
    gk = torch.rand(300, generator=g).cuda()
    one, two = kd_grads(h, W, y, ids, z, tau, gk, gk), kd_grads(h, W, y, ids, z, tau, gk, gk.clone())
    assert torch.equal(one[0], two[0]) and torch.equal(one[1], two[1])


def near_or_past(got, want, what):
    """near, or an infinity of the value's sign where the value may be past the type's largest (bf16's is 3.39e38; with
    weights of 3.5e38 in all, an element of dW is 3.81e38)."""
    ref, err = want
    over = got.isinf() & (ref.abs() + err + 2.0 ** -8 * (ref.abs() + err) >= torch.finfo(got.dtype).max)
    assert torch.equal(got[over] > 0, ref[over] > 0)
    near(torch.where(over, 0, got), (torch.where(over, 0, ref), err), what, 2.0 ** -8)


@pytest.mark.parametrize("small,large", [(1e-30, 1e10), (1e-20, 1e15), (1e-4, 1e8), (1e-38, 1e38)])
def test_losses_of_very_different_weights(small, large):
    """One loss's weights may be any size beside the other's: the larger one's gradient where a token has both, and the
    smaller one's (to 1e-30 at least) where it has only that."""
    n, V, d = 60, 270, 64
    h, W, y, g = inputs(n, V, d, seed=9)
    ids, z = teacher(n, V, 6, g)
    gk, gc = torch.randn(n, generator=g).cuda(), torch.randn(n, generator=g).cuda()
    want = oracle(h, W, y, small * gc, None, ids, z, 2.0, large * gk)
    got = kd_grads(h, W, y, ids, z, 2.0, large * gk, small * gc)
    near_or_past(got[0], want["dh"], "dh"), near_or_past(got[1], want["dW"], "dW")
    a, b = h.clone().requires_grad_(), W.clone().requires_grad_()
    got = torch.autograd.grad(linear_cross_entropy(a, b, y), (a, b), (small * gc, large * gk))
    want = oracle(h, W, y, small * gc, large * gk)
    near_or_past(got[0], want["dh"], "dh"), near_or_past(got[1], want["dW"], "dW")


@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_teacher_taken_out_of_the_loss(bad):
    """A token whose teacher is no distribution (its loss is NaN), its weight zero: the gradients of the token's cross
    entropy, and of all other tokens, are those with any finite logits there."""
    n, V, d = 40, 90, 64
    h, W, y, g = inputs(n, V, d, seed=10, pad=0)
    ids = torch.stack([torch.randperm(V, generator=g)[:7] for _ in range(n)]).cuda()
    z = torch.randn(n, 7, generator=g).cuda()
    keep = torch.arange(n, device="cuda") % 4 != 1
    gk, gc = torch.randn(n, generator=g).cuda(), torch.randn(n, generator=g).cuda()
    worse = z.clone()
    worse[1::4, 2] = bad
    for tau in (1.0, 2.0):
        grads = []
        for logits in (z, worse):
            a, b = h.clone().requires_grad_(), W.clone().requires_grad_()
            kd, ce = linear_distill(a, b, ids, logits, tau, y)
            loss = (torch.where(keep, kd, 0) * gk + ce * gc).sum()
            assert torch.isfinite(loss)
            grads.append(torch.autograd.grad(loss, (a, b)))
        assert all(torch.equal(p, q) and torch.isfinite(p).all() for p, q in zip(*grads))
        want = oracle(h, W, y, gc, None, ids, z, tau, torch.where(keep, gk, 0))
        near(grads[1][0], want["dh"], "dh", 2.0 ** -8), near(grads[1][1], want["dW"], "dW", 2.0 ** -8)


@pytest.mark.parametrize("n", [32768, 32769, 70001])
def test_many_tokens(n):
    """The scale over more tokens than one workgroup looks at: padding's weights have no say, one large weight (the last
    token's, a workgroup's first or last) does."""
    V, d = 40, 16
    h, W, y, g = inputs(n, V, d, seed=11, pad=0.2)
    for at in (0, 255, 256, 1023, n - 1, None):
        gc = 1e-4 * torch.rand(n, generator=g).cuda()
        if at is not None:
            y[at], gc[at] = 7, -3.0
        here = torch.where(y >= 0, gc, 0)
        want = ce_grads(h, W, y, here)
        for a, b in zip(ce_grads(h, W, y, torch.where(y >= 0, gc, 3e38)), want):
            assert torch.equal(a, b)
        ref = oracle(h, W, y, here)
        near(want[2], ref["dh"], "dh", 2.0 ** -8), near(want[3], ref["dW"], "dW", 2.0 ** -8)
