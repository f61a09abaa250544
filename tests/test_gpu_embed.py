"""The token lookup with a scale and its gradient by sorted tokens, against plain forms in 64 bits.

Tolerances: a row is one fp32 product rounded to its type (2^-24 and half a step of the type); a gradient row sums m
terms in fp32 (at most m 2^-24 of the sum of magnitudes), is scaled and rounded to its type."""
import pytest
import torch

from pragnosia_amd.embed import embedding

pytestmark = pytest.mark.gpu
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}
f32, b16 = torch.float32, torch.bfloat16


def make_ids(kind, n, V, g):
    if kind == "uniform":
        return torch.randint(0, V, (n,), generator=g)
    if kind == "one":
        return torch.full((n,), V - 1)
    if kind == "zipf":
        return ((float(V) ** torch.rand(n, generator=g)).long() - 1).clamp(0, V - 1)
    if kind == "none":
        return torch.where(torch.rand(n, generator=g) < 0.5, -1, V + 5)
    ids = torch.randint(-2, V + 2, (n,), generator=g)  # "padded"
    ids[: n // 2] = torch.randint(0, max(1, V // 100), (n // 2,), generator=g)
    return ids


def check(ids, V, d, wt, yt, gt_scale=1.0, scale=1.7, seed=0):
    g = torch.Generator().manual_seed(seed)
    W = torch.randn(V, d, generator=g).to(wt).cuda().requires_grad_()
    ids = ids.cuda()
    y = embedding(ids, W, scale, yt)
    on = (ids >= 0) & (ids < V)
    s32 = float(torch.tensor(scale, dtype=f32))
    want = torch.where(on[..., None], W.detach().double()[ids.clamp(0, V - 1)] * s32, 0)
    assert y.dtype == yt and y.shape == (*ids.shape, d)
    assert ((y.double() - want).abs() <= (HALF[yt] + 2.0 ** -24) * want.abs()).all()
    gy = torch.randn(y.shape, generator=g).to(yt).cuda()
    dW, = torch.autograd.grad(y, W, gy)
    assert dW.dtype == wt and dW.shape == W.shape
    flat, gf = ids.reshape(-1).long(), gy.reshape(-1, d).double() * on.reshape(-1, 1)
    at = flat.clamp(0, V - 1)
    ref = torch.zeros(V, d, device="cuda", dtype=torch.float64).index_add_(0, at, gf) * s32
    size = torch.zeros(V, d, device="cuda", dtype=torch.float64).index_add_(0, at, gf.abs()) * abs(s32)
    m = torch.bincount(at[on.reshape(-1)], minlength=V)[:, None].double()
    bound = (m + 2) * 2.0 ** -24 * size + HALF[wt] * (ref.abs() + (m + 2) * 2.0 ** -24 * size)
    off = (dW.double() - ref).abs() - bound
    assert (off <= 0).all(), off.max()
    assert not dW[m[:, 0] == 0].any()
    again, = torch.autograd.grad(embedding(ids, W, scale, yt), W, gy)
    assert torch.equal(again, dW)  # one order, one result


@pytest.mark.parametrize("kind", ["uniform", "one", "zipf", "none", "padded"])
@pytest.mark.parametrize("n,V,d", [(1, 1, 8), (33, 5, 8), (100, 40, 72), (1000, 257, 264), (5000, 20011, 64)])
def test_values_and_gradient(kind, n, V, d):
    g = torch.Generator().manual_seed(n + V)
    check(make_ids(kind, n, V, g), V, d, f32, f32)


@pytest.mark.parametrize("wt,yt", [(b16, b16), (f32, b16), (b16, f32)])
def test_types(wt, yt):
    g = torch.Generator().manual_seed(1)
    check(make_ids("padded", 700, 90, g), 90, 136, wt, yt)


@pytest.mark.parametrize("kind", ["one", "zipf"])
def test_long_runs(kind):
    """A word that is most of a long batch: the whole order in one id's run, and in runs of every length."""
    g = torch.Generator().manual_seed(2)
    check(make_ids(kind, 70001, 1500, g).view(1, -1), 1500, 24, f32, f32)
