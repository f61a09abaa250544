"""Rows times a 4-bit weight where there are too many tiles for the kernel of few: every form of the tiled kernel with every
epilogue, norms, numbers that are not finite, contracted axes of many chunks, repeats and replays."""
import math

import pytest
import torch

from pragnosia_amd import fp4

from test_gpu_fp4 import BF16, F32, check, layer_norm, rows, weight

pytestmark = pytest.mark.gpu
DEV = "cuda"

# (rows, columns) of each form, the columns whole vectors or not. Tiles of 16 x 16 past 256 of them leave the kernel of few;
# then 16 x 64, 32 x 128 and 32 x 256 in one round of workgroups, and 32 x 256 in several
FORMS = {"16x64": (32, 2320), "16x64 ragged": (41, 2321), "32x128": (100, 2400), "32x128 ragged": (97, 2407),
         "32x256": (330, 3016), "32x256 ragged": (330, 3013), "32x256 rounds": (1000, 2200), "32x256 rounds ragged": (1001, 2203)}
forms = pytest.mark.parametrize("form", list(FORMS))
# 9 to 15 blocks of 128 columns, the last cut short: odd and even numbers of chunks of one, two and four blocks, more than two
DEPTHS = (1160, 1400, 1800)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("group", [32, 64, 128])
@forms
def test_epilogues(form, group, dtype):
    n, N = FORMS[form]
    for i, K in enumerate(DEPTHS):
        Q = fp4.quantize(weight(N, K, dtype, seed=K), group)
        x, b, r = rows(n, K, dtype, K + 1), rows(1, N, dtype, 3)[0], rows(n, N, dtype, 4)
        if i == 0:
            check(x, Q, act="gelu")
            check(x, Q, resid=r, norm=layer_norm(K, dtype, bias=False))
        elif i == 1:
            check(x, Q, bias=b, act="gelu", resid=r)
            check(x, Q, bias=b, act="gelu", norm=layer_norm(K, dtype))
        else:
            check(x, Q, bias=b, act="gelu", resid=r, norm=layer_norm(K, dtype))
            check(x, Q, bias=b, norm=layer_norm(K, dtype, bias=False))


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("n,N", [(960, 4096), (959, 4099)])
def test_epilogues_of_the_largest_tiles(n, N, group):
    """64 x 256, of bf16 rows without a norm along an axis of 2048 or more: 8 and 9 chunks."""
    for K in (2048, 2184):
        Q = fp4.quantize(weight(N, K, BF16), group)
        x, b, r = rows(n, K, BF16), rows(1, N, BF16, 3)[0], rows(n, N, BF16, 4)
        check(x, Q, act="gelu")
        check(x, Q, bias=b, act="gelu", resid=r)


@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("dtype", [F32, BF16])
@forms
def test_not_finite(form, dtype, norm):
    """An infinity or a NaN in a row stays in that row's results."""
    n, N = FORMS[form]
    K = 1160
    Q = fp4.quantize(weight(N, K, dtype), 64)
    x, ln = rows(n, K, dtype), layer_norm(K, dtype) if norm else None
    clean = fp4.linear(x, Q, norm=ln)
    at = n // 2
    others = torch.arange(n, device=DEV) != at
    x[at, 7], x[at, K - 1] = math.inf, math.inf
    got = fp4.linear(x, Q, norm=ln)
    assert torch.equal(got[others], clean[others])
    if norm:
        assert got[at].isnan().all()  # (the row's mean)
    else:
        want = (x[at].float() * fp4.dequantize(Q, F32)).sum(1)
        assert torch.equal(got[at].isnan(), want.isnan()) and not got[at].isfinite().any()
        assert torch.equal(got[at] == math.inf, want == math.inf) and torch.equal(got[at] == -math.inf, want == -math.inf)
    x[at, 7] = math.nan
    got = fp4.linear(x, Q, norm=ln)
    assert got[at].isnan().all() and torch.equal(got[others], clean[others])


@pytest.mark.parametrize("dtype", [F32, BF16])
@forms
def test_same_bits(form, dtype):
    """The same call gives the same bits, and a row's do not depend on the others of its kind of block."""
    n, N = FORMS[form]
    Q, ln = fp4.quantize(weight(N, 1400, dtype), 64), layer_norm(1400, dtype)
    x = rows(n, 1400, dtype)
    for kw in ({}, dict(norm=ln, act="gelu")):
        a = fp4.linear(x, Q, **kw)
        assert all(torch.equal(fp4.linear(x, Q, **kw), a) for _ in range(3))
        assert torch.equal(fp4.linear(x.flip(0), Q, **kw).flip(0), a)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("form", [f for f in FORMS if "ragged" not in f])
def test_graph(form, dtype):
    """Captured with the weight's rounding, replayed with eager work between."""
    n, N = FORMS[form]
    K = 1160
    ln, buf, W = layer_norm(K, dtype), rows(n, K, dtype), weight(N, K, dtype)
    fp4.linear(buf, fp4.quantize(W, 64), norm=ln, act="gelu")
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        R = fp4.quantize(W, 64)
        y, plain = fp4.linear(buf, R, norm=ln, act="gelu"), fp4.linear(buf, R)
    for seed in (11, 12, 13):
        buf.copy_(rows(n, K, dtype, seed))
        W.copy_(weight(N, K, dtype, seed))
        g.replay()
        torch.cuda.synchronize()
        Q = fp4.quantize(W, 64)
        assert torch.equal(y, fp4.linear(buf, Q, norm=ln, act="gelu")) and torch.equal(plain, fp4.linear(buf, Q))
