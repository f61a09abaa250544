"""A normalised bf16 row keeps its 32 bits into the product with a 4-bit weight: seen where a residual takes the product's
leading bits away."""
import pytest
import torch

from pragnosia_amd import fp4

pytestmark = pytest.mark.gpu
DEV = "cuda"
F64 = torch.float64


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("n,N", [(1, 40), (4, 40), (16, 40), (21, 4100), (70, 4100), (300, 4100), (1000, 4100)])
def test_normalised_bf16_row_is_not_rounded(n, N, group):
    """Row j of the weight holds one 6 (a code and a scale without error), so the product is 6 z of one normalised value, and
    the residual is minus that rounded to bf16.

    z is off by what its mean, 1 / sigma and the three operations on it are, each chain of K / 128 + 16 additions by 2^-23 a
    step; the product's sum by one step of 2^-23 for each part that z is given in; the result's rounding is 2^-8 of the
    little that is left. Sixteen bits of z would be off by up to 2^-15 of it."""
    K = 264
    g = torch.Generator().manual_seed(n + group)
    x = torch.randn(n, K, generator=g).bfloat16().to(DEV)
    norm = torch.nn.LayerNorm(K, device=DEV, dtype=torch.bfloat16).requires_grad_(False)
    norm.weight.copy_(1 + 0.2 * torch.randn(K, generator=g))
    norm.bias.copy_(0.2 * torch.randn(K, generator=g))
    col = torch.arange(N, device=DEV) * 7 % K
    W = torch.zeros(N, K, device=DEV, dtype=torch.bfloat16)
    W[torch.arange(N, device=DEV), col] = 6.0
    Q = fp4.quantize(W, group)
    assert torch.equal(fp4.dequantize(Q), W)

    v = x.to(F64)
    rstd = (v.var(1, unbiased=False, keepdim=True) + norm.eps).rsqrt()
    hat, gain = (v - v.mean(1, keepdim=True)) * rstd, norm.weight.to(F64)
    z = hat * gain + norm.bias.to(F64)
    chain = (K / 128 + 16) * 2.0 ** -23
    off = (gain.abs() * rstd * chain * v.abs().mean(1, keepdim=True) * (1 + hat.abs())
           + gain.abs() * hat.abs() * (chain + 2.0 ** -21) + z.abs() * 2.0 ** -22)
    y, off = 6 * z[:, col], 6 * off[:, col]
    off = off + 3 * 2.0 ** -23 * y.abs()
    resid = -y.bfloat16()
    want = y + resid.to(F64)
    got = fp4.linear(x, Q, norm=norm, resid=resid).to(F64)
    bound = off * (1 + 2.0 ** -8) + 2.0 ** -8 * want.abs()
    assert ((got - want).abs() <= bound).all(), f"{((got - want).abs() / bound).max().item():.3g} of the bound"
