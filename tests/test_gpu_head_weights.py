"""The head's gradients under the per-token weights that autograd hands back: weights of tokens that have no say, of
very different sizes, the same tensor for both losses, and a token taken out of one loss only."""
import math

import pytest
import torch

from pragnosia_amd.head import linear_distill
from test_gpu_head import ce_grads, inputs, near, oracle, teacher

pytestmark = pytest.mark.gpu
SIZES = [1e30, 3e38, math.inf, math.nan]


def kd_grads(h, W, y, ids, z, tau, g_kd, g_ce=None):
    a, b = h.detach().clone().requires_grad_(), W.detach().clone().requires_grad_()
    kd, ce = linear_distill(a, b, ids, z, tau, y)
    return torch.autograd.grad(kd if y is None else (kd, ce), (a, b), g_kd if y is None else (g_kd, g_ce))


@pytest.mark.parametrize("tau", [1.0, 3.0])
def test_one_weight_tensor_for_both_losses(tau):
    """The weights of the two losses in one tensor, or in two of equal values: the same bits."""
    h, W, y, g = inputs(300, 270, 64, seed=8)
    ids, z = teacher(300, 270, 6, g)
    gk = torch.rand(300, generator=g).cuda()
    one, two = kd_grads(h, W, y, ids, z, tau, gk, gk), kd_grads(h, W, y, ids, z, tau, gk, gk.clone())
    assert torch.equal(one[0], two[0]) and torch.equal(one[1], two[1])
