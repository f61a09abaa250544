"""4-bit weights against the definition in 64 bits: rounding (every code, ties, odd sizes, zeros, the smallest and largest
scales, infinities), the layout, reading back, and rows times such a weight."""
import math

import pytest
import torch

from pragnosia_amd import fp4
from pragnosia_amd._lib import PragnosiaError

pytestmark = pytest.mark.gpu
DEV = "cuda"
E2M1 = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)
F32, BF16 = torch.float32, torch.bfloat16


def scales_of(W, group):
    """(N, groups) fp64, from the definition: max |w| / 6 rounded to fp32, then bf16."""
    N, K = W.shape
    a = torch.nn.functional.pad(W.double().abs(), (0, -K % group)).view(N, -1, group).amax(2)
    s = (a / 6).float().bfloat16().double()
    return torch.where(a.isfinite(), s, math.nan)


def rounded(W, group):
    """The weight that W is rounded to, fp64 on the CPU: among the values s v the nearest, an even code in a tie."""
    W = W.detach().cpu()
    N, K = W.shape
    s = scales_of(W, group).repeat_interleave(group, 1)[:, :K]
    w = W.double()
    away = (w.abs()[..., None] - E2M1 * s[..., None]).abs()
    near = away.amin(-1, keepdim=True)
    even = (torch.arange(8) % 2 == 0).expand(away.shape)
    pick = torch.where(away == near, torch.where(even, 2, 1), 0).argmax(-1)
    v = torch.copysign(E2M1[pick] * s, w)
    return torch.where(s.isnan(), math.nan, torch.where(s == 0, 0.0, v))


def weight(N, K, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(N, K, generator=g) * torch.randn(N, 1, generator=g).exp()).to(dtype).to(DEV)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("N,K", [(1, 8), (16, 128), (17, 136), (5, 1000), (130, 328), (33, 24)])
def test_rounding(N, K, group, dtype):
    W = weight(N, K, dtype)
    got = fp4.dequantize(fp4.quantize(W, group), F32).double().cpu()
    assert torch.equal(got, rounded(W, group))


@pytest.mark.parametrize("group", [32, 64, 128])
def test_ties_and_borders(group):
    """Every border between two codes, exactly and one fp32 step to either side, at scales that bf16 rounded up and down
    and at the smallest and largest."""
    mids = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], dtype=torch.float64)
    rows = []
    for top in (6.0, 5.99, 6.03, 1.7e-3, 8.1e-36, 3.3e-38, 2.0e-39, 1.2e-42, 3.0e38, 1.1e31):
        s = torch.tensor(top, dtype=F32).double().div(6).float().bfloat16().double()
        t = (mids * s).float()
        near = torch.cat([t, torch.nextafter(t, t.new_full((), math.inf)), torch.nextafter(t, t.new_full((), 0.0))])
        row = torch.zeros(32)
        row[:21], row[21] = near, top
        row[22:25] = -t[:3]
        row[25] = -0.0
        rows.append(row.repeat(group // 32))
    W = torch.stack(rows).to(DEV)
    got = fp4.dequantize(fp4.quantize(W, group), F32).double().cpu()
    assert torch.equal(got, rounded(W, group))


def test_groups_of_zeros_and_not_finite():
    W = weight(20, 256, F32)
    W[3, :64] = 0.0
    W[4, 70], W[5, 200], W[6, 0] = math.inf, -math.inf, math.nan
    got = fp4.dequantize(fp4.quantize(W, 64), F32).double().cpu()
    assert torch.equal(got.nan_to_num(7e9), rounded(W, 64).nan_to_num(7e9))
    assert got[4].isnan().sum() == got[5].isnan().sum() == got[6].isnan().sum() == 64 and got.isnan().sum() == 192
    assert (got[3, :64] == 0).all()
    # such a group makes its row NaN and no other
    y = fp4.linear(torch.ones(3, 256, device=DEV), fp4.quantize(W, 64))
    assert torch.equal(y.isnan().any(0).nonzero().flatten().cpu(), torch.tensor([4, 5, 6]))


@pytest.mark.parametrize("group", [32, 64, 128])
def test_layout(group):
    """Codes and scales lie as the header says; what is past the edge is zero."""
    N, K = 21, 200
    W = weight(N, K, F32)
    Q = fp4.quantize(W, group)
    rt, kb = 2, 2
    words = Q.codes.cpu().view(rt, kb, 64, 16)
    codes = torch.zeros(rt * 16, kb * 128, dtype=torch.long)
    for lane in range(64):
        for byte in range(16):
            j, e = byte // 4, byte % 4 * 2
            for half in range(2):
                col = 32 * j + 8 * (lane // 16) + e + half
                for a in range(rt):
                    for b in range(kb):
                        codes[16 * a + lane % 16, 128 * b + col] = words[a, b, lane, byte] >> 4 * half & 15
    scales = Q.scales.cpu().double().view(rt, kb, 16, -1).permute(0, 2, 1, 3).reshape(rt * 16, -1)
    v = E2M1[codes & 7] * torch.where(codes >= 8, -1.0, 1.0) * scales.repeat_interleave(group, 1)
    assert torch.equal(v[:N, :K], rounded(W, group))
    assert not codes[N:].any() and not codes[:, K:].any() and not scales[N:].any()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_read_back_rounds_once(dtype):
    W = weight(70, 264, BF16)
    Q = fp4.quantize(W, 32)
    assert Q.dtype == BF16 and Q.shape == (70, 264) and Q.nbytes == Q.codes.numel() + 2 * Q.scales.numel()
    assert torch.equal(fp4.dequantize(Q, dtype).cpu(), rounded(W, 32).to(dtype))


def test_views_and_out():
    big = weight(64, 528, F32)
    want = rounded(big[1:64:2, 8:400].contiguous(), 64)
    assert torch.equal(fp4.dequantize(fp4.quantize(big[1:64:2, 8:400], 64)).double().cpu(), want)
    assert torch.equal(fp4.dequantize(fp4.quantize(big.t()[:, :32], 32)).double().cpu(), rounded(big.t()[:, :32], 32))
    Q = fp4.quantize(torch.zeros(32, 392, device=DEV), 64)
    at = Q.codes.data_ptr()
    assert fp4.quantize(big[1:64:2, 8:400], 64, out=Q) is Q and Q.codes.data_ptr() == at
    assert torch.equal(fp4.dequantize(Q).double().cpu(), want)
    P = torch.nn.Parameter(big)
    assert not fp4.dequantize(fp4.quantize(P)).requires_grad


# ---------------------------------------------------------------------------------------------------------------
# rows times a weight

def linear64(x, Q, bias=None, norm=None, act=None, resid=None):
    """The result in 64 bits and a bound of the error of one computed in fp32 from x's type: (y, bound).

    A product's parts are exact, and a sum of K of them is a chain of at most K / 8 + 24 fp32 additions, each off by at most
    2^-23 of the sum of absolute values (matrix instructions may cut where an addition would round). A normalised value is
    off by a few steps of what it was formed from; a bf16 row's is kept to 16 bits."""
    W = fp4.dequantize(Q, F32).double()
    z, dz = x.double(), torch.zeros_like(x, dtype=torch.float64)
    K = W.shape[1]
    if norm is not None:
        mean, var = z.mean(1, keepdim=True), z.var(1, unbiased=False, keepdim=True)
        rstd = (var + norm.eps).rsqrt()
        g = norm.weight.double()
        hat = (z - mean) * rstd
        # the mean is off by its sum's rounding, and 1 / sigma by the squares' sum and this; each at most 2^-23 times a
        # chain of K / 128 + 16 additions
        chain = (K / 128 + 16) * 2.0 ** -23
        dz = (g.abs() * rstd * chain * z.abs().mean(1, keepdim=True) * (1 + hat.abs())
              + g.abs() * hat.abs() * (chain + 2.0 ** -21))
        z = hat * g
        if norm.bias is not None:
            z = z + norm.bias.double()
        dz = dz + z.abs() * 2.0 ** -22
        if x.dtype == BF16:
            dz = dz + z.abs() * 2.0 ** -15
    y = z @ W.t()
    bound = (K / 8 + 24) * 2.0 ** -23 * (z.abs() @ W.abs().t()) + dz @ W.abs().t()
    if bias is not None:
        y = y + bias.double()
        bound = bound + 2.0 ** -23 * y.abs()
    if act == "gelu":
        y = torch.nn.functional.gelu(y)
        bound = 1.13 * bound + 2.0 ** -20 * y.abs() + 2.0 ** -22  # |gelu'| < 1.13; erff within a few steps of 1
    if resid is not None:
        y = y + resid.double()
    eps = 2.0 ** -8 if x.dtype == BF16 else 2.0 ** -23
    return y, bound * (1 + eps) + eps * y.abs() + 1e-37


def check(x, Q, **kw):
    got = fp4.linear(x, Q, kw.get("bias"), norm=kw.get("norm"), act=kw.get("act"), resid=kw.get("resid"))
    assert got.dtype == x.dtype and got.shape == (x.shape[0], Q.N)
    want, bound = linear64(x, Q, **kw)
    off = (got.double() - want).abs()
    assert (off <= bound).all(), f"{(off / bound).max().item():.3g} of the bound"
    return got


def rows(n, K, dtype, seed=1):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(n, K, generator=g).to(dtype).to(DEV)


def layer_norm(K, dtype, bias=True):
    m = torch.nn.LayerNorm(K, device=DEV, dtype=dtype, bias=bias).requires_grad_(False)
    g = torch.Generator().manual_seed(2)
    m.weight.copy_(1 + 0.2 * torch.randn(K, generator=g))
    if bias:
        m.bias.copy_(0.2 * torch.randn(K, generator=g))
    return m


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("n", [1, 2, 4, 5, 16, 17, 33, 64, 65, 100, 257])
def test_linear_rows(n, group, dtype):
    """Every kind of row block, with an odd number of outputs and a short last group."""
    Q = fp4.quantize(weight(77, 328, dtype), group)
    check(rows(n, 328, dtype), Q)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n", [1, 3, 16, 70])
@pytest.mark.parametrize("N,K", [(1, 8), (15, 24), (16, 128), (1030, 704), (40, 2056), (100, 4104), (24, 8192)])
def test_linear_sizes(N, K, n, dtype):
    Q = fp4.quantize(weight(N, K, dtype), 64)
    check(rows(n, K, dtype), Q)
    check(rows(n, K, dtype), Q, norm=layer_norm(K, dtype))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("n,N,K", [(21, 1000, 264), (21, 4100, 264), (70, 4100, 264), (300, 4100, 264), (1000, 4100, 264),
                                   (959, 4100, 2056), (960, 4096, 2048), (1024, 4096, 2048)])
def test_linear_tiles(n, N, K, group, dtype):
    """Numbers of rows and columns that ask for ever larger tiles, whole and with ragged edges."""
    Q = fp4.quantize(weight(N, K, dtype), group)
    bias, resid = rows(1, N, dtype, 4)[0], rows(n, N, dtype, 5)
    check(rows(n, K, dtype), Q, bias=bias, resid=resid)
    check(rows(n, K, dtype), Q, norm=layer_norm(K, dtype))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n", [1, 4, 6, 90])
def test_linear_epilogue(n, dtype):
    N, K = 200, 512
    Q = fp4.quantize(weight(N, K, dtype), 128)
    x, b, r = rows(n, K, dtype), rows(1, N, dtype, 3)[0], rows(n, N, dtype, 4)
    check(x, Q, bias=b)
    check(x, Q, act="gelu")
    check(x, Q, resid=r)
    check(x, Q, bias=b, act="gelu", resid=r, norm=layer_norm(K, dtype))
    check(x, Q, bias=b, resid=r, norm=layer_norm(K, dtype, bias=False))


@pytest.mark.parametrize("n", [1, 3, 20])
def test_linear_is_fp32(n):
    """fp32 rows are not rounded: rows of 2^0 and 2^-20 beside each other, and rows far from zero before a norm."""
    Q = fp4.quantize(weight(64, 768, F32), 64)
    x = rows(n, 768, F32)
    x[:, ::2] *= 2.0 ** -20
    check(x, Q)
    check(rows(n, 768, F32) * 0.5 + 40.0, Q, norm=layer_norm(768, F32))


@pytest.mark.parametrize("n", [1, 4, 40, 80])
def test_linear_not_finite(n):
    """An infinity or a NaN in a row stays in that row's results, as in an fp32 product."""
    Q = fp4.quantize(weight(48, 256, F32), 64)
    x = rows(n, 256, F32)
    clean = fp4.linear(x, Q)
    x[n // 2, 7], x[n // 2, 9] = math.inf, math.inf
    got, W = fp4.linear(x, Q), fp4.dequantize(Q)
    want = (x[n // 2] * W).sum(1)
    assert torch.equal(got[n // 2].isnan(), want.isnan()) and torch.equal(got[n // 2] == math.inf, want == math.inf)
    assert torch.equal(got[n // 2] == -math.inf, want == -math.inf) and not got[n // 2].isfinite().any()
    others = torch.arange(n, device=DEV) != n // 2
    assert torch.equal(got[others], clean[others])
    x[n // 2, 9] = torch.tensor(0x7f800001, dtype=torch.int32).view(F32)  # a NaN whose upper half is an infinity's
    assert fp4.linear(x, Q)[n // 2].isnan().all()


def test_linear_same_bits_and_rows_alone():
    Q = fp4.quantize(weight(300, 768, F32), 64)
    x = rows(40, 768, F32)
    a = fp4.linear(x, Q)
    assert all(torch.equal(fp4.linear(x, Q), a) for _ in range(3))
    assert torch.equal(fp4.linear(x[:20], Q), a[:20])  # (the same kind of row block)


def test_linear_shapes_views_and_types():
    Q = fp4.quantize(weight(96, 256, F32), 64)
    x = rows(6, 256, F32)
    want = fp4.linear(x, Q)
    assert torch.equal(fp4.linear(x.view(2, 3, 256), Q), want.view(2, 3, 96))
    assert fp4.linear(x[0], Q).shape == (96,) and fp4.linear(x[:0], Q).shape == (0, 96)
    wide = rows(6, 520, F32)
    wide[:, 3:259] = x
    assert torch.equal(fp4.linear(wide[:, 3:259], Q), want)  # strided, and not at a 16-byte address
    assert torch.equal(fp4.linear(x.t().contiguous().t(), Q), want)
    b = rows(1, 96, BF16, 5)[0]
    assert torch.equal(fp4.linear(x, Q, b), fp4.linear(x, Q, b.float()))  # operands of another type are converted
    r = rows(6, 97, F32)[:, 1:]
    assert torch.equal(fp4.linear(x, Q, resid=r), fp4.linear(x, Q, resid=r.contiguous()))


def test_linear_streams_and_graph():
    Q = fp4.quantize(weight(500, 768, F32), 64)
    x, ln = rows(9, 768, F32), layer_norm(768, F32)
    want = fp4.linear(x, Q, norm=ln, act="gelu")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = fp4.linear(x, Q, norm=ln, act="gelu")
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    buf, W = x.clone(), weight(500, 768, F32)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        R = fp4.quantize(W, 64)
        y = fp4.linear(buf, R, norm=ln, act="gelu")
    for seed in (11, 12, 13):
        buf.copy_(rows(9, 768, F32, seed))
        W.copy_(weight(500, 768, F32, seed))
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, fp4.linear(buf, fp4.quantize(W, 64), norm=ln, act="gelu"))


def test_linear_refuses_gradients():
    Q = fp4.quantize(weight(32, 64, F32), 32)
    x = rows(2, 64, F32).requires_grad_()
    with pytest.raises(PragnosiaError, match="no backward"):
        fp4.linear(x, Q)
    with torch.no_grad():
        fp4.linear(x, Q)


def test_linear_trace():
    """make_fx and a compiled call see the custom op; the results are the eager call's."""
    from torch.fx.experimental.proxy_tensor import make_fx
    Q = fp4.quantize(weight(48, 128, F32), 32)
    x, ln, b = rows(5, 128, F32), layer_norm(128, F32), rows(1, 48, F32, 3)[0]
    f = lambda x: fp4.linear(x, Q, b, norm=ln, act="gelu")  # noqa: E731
    traced = make_fx(f)(x)
    assert "fp4_linear" in traced.code and torch.equal(traced(x), f(x))
    torch.library.opcheck(torch.ops.pragnosia_gen.fp4_linear.default,
                          (x, Q.codes, Q.scales, ln.weight, ln.bias, 1e-5, b, 1, None, 48, 32),
                          test_utils=("test_schema", "test_faketensor"))
    torch.library.opcheck(torch.ops.pragnosia_gen.fp4_quantize.default, (weight(40, 72, F32), 64),
                          test_utils=("test_schema", "test_faketensor"))


def test_large_offsets():
    """More than 2^31 codes: the last rows' tiles lie past 2^30 bytes, the weight's past 2^32."""
    N, K = 1 << 18, 8200
    W = torch.zeros(N, K, device=DEV, dtype=BF16)
    tail = weight(100, K, BF16)
    W[-100:] = tail
    Q = fp4.quantize(W, 128)
    del W
    last = fp4.quantize(tail, 128)
    x = rows(2, K, BF16)
    y = fp4.linear(x, Q)
    assert not y[:, :-112].any() and torch.equal(y[:, -100:], fp4.linear(x, last))
    back = fp4.dequantize(Q, BF16)
    assert torch.equal(back[-100:], fp4.dequantize(last, BF16)) and not back[:-100].any()
