"""GPU: the LM class's losses with fused_ends take what the model without it takes."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_targets_of_any_layout():
    """Targets (B, T), flat, or a slice of longer sequences beside hidden rows (B, T, d): one loss, to the bit, and that
    of the model without the switch to the rounding of its logits (bf16: 2^-8 of the largest, each way)."""
    from pragnosia_amd.model import LM
    losses = {}
    for fused in (False, True):
        torch.manual_seed(0)
        with torch.device("cuda"):
            m = LM(vocab=503, d=64, layers=1, mlp_mult=1, ctx=40, fused_ends=fused)
        g = torch.Generator(device="cuda").manual_seed(1)
        xs = torch.randint(0, 503, (3, 41), generator=g, device="cuda")
        h = torch.randn(3, 40, 64, generator=g, device="cuda")
        y = xs[:, 1:]
        losses[fused] = [m.loss(h, y), m.loss(h, y.reshape(-1)), m.loss(h.reshape(-1, 64), y.reshape(-1)),
                         m.loss(h, y.contiguous().view(3 * 40, 1))]
        assert all(torch.equal(a, losses[fused][0]) for a in losses[fused])
        top = (h.reshape(-1, 64) @ m.e.weight.t()).abs().max()
    assert abs(losses[True][0] - losses[False][0]) <= 2.0 ** -7 * top
