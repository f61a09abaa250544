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
@pytest.mark.parametrize("n,V,d", [(1, 1, 8), (33, 5, 8), (100, 40, 72), (256, 100, 264), (257, 100, 264),
                                   (1000, 257, 264), (5000, 20011, 64)])
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


@pytest.mark.parametrize("n", [3000, 20000])
def test_many_ids_of_one_range(n):
    """Tokens of some tens of neighbouring ids in a large table: many ids among a wave's tokens, more than its list."""
    g = torch.Generator().manual_seed(6)
    check(torch.randint(100, 164, (n,), generator=g), 20000, 16, f32, f32)


def test_strides_offsets_and_shapes():
    """ids of any shape and integer type, a table inside a larger buffer at an odd offset, an expanded gradient."""
    g = torch.Generator().manual_seed(3)
    W = torch.randn(50 * 16 + 1, generator=g).cuda()[1:].view(50, 16).requires_grad_()
    assert W.data_ptr() % 16
    ids = torch.randint(0, 50, (7, 2, 3), generator=g).cuda()
    dense = W.detach().clone().requires_grad_()
    want, = torch.autograd.grad(embedding(ids.permute(2, 0, 1).reshape(-1), dense, 2.0).sum(), dense)
    for t in (ids.permute(2, 0, 1), ids.permute(2, 0, 1).int(), ids.permute(2, 0, 1).to(torch.uint8)):
        y = embedding(t, W, 2.0)
        assert y.shape == (3, 7, 2, 16) and torch.equal(y, 2 * W[t.long()])
        assert torch.equal(torch.autograd.grad(y.sum(), W)[0], want)
    assert torch.equal(embedding(torch.tensor(3, device="cuda"), W), W[3])


def test_nothing_to_do():
    W = torch.randn(5, 8, device="cuda", requires_grad=True)
    y = embedding(torch.zeros(0, 4, dtype=torch.long, device="cuda"), W)
    assert y.shape == (0, 4, 8)
    dW, = torch.autograd.grad(y.sum(), W)
    assert dW.shape == W.shape and not dW.any()


def test_infinities_stay_in_their_rows():
    """A NaN or infinity in one token's gradient reaches its own id's row and no other; in a padding token's, none."""
    ids = torch.tensor([3, 1, 3, -1, 7] * 9, device="cuda")
    W = torch.zeros(9, 8, device="cuda", requires_grad=True)
    gy = torch.ones(45, 8, device="cuda")
    gy[3::5] = float("nan")
    gy[1] = float("inf")
    dW, = torch.autograd.grad(embedding(ids, W), W, gy)
    assert torch.equal(dW[[0, 3, 7]], torch.tensor([0.0, 18.0, 9.0], device="cuda")[:, None].expand(3, 8))
    assert torch.isinf(dW[1]).all()


def test_streams_and_capture():
    """Two gradients at once on streams of their own, and one captured and replayed on new ids: the eager bits."""
    g = torch.Generator().manual_seed(4)
    W = torch.randn(700, 64, generator=g).cuda().requires_grad_()
    ids = [make_ids("zipf", n, 700, g).cuda() for n in (5000, 3000)]
    gy = [torch.randn(i.shape[0], 64, generator=g).cuda() for i in ids]

    def grad(i, q):
        return torch.autograd.grad(embedding(i, W, 0.5), W, q)[0]

    want = [grad(i, q) for i, q in zip(ids, gy)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in ids]
    got = []
    for s, i, q in zip(streams * 3, ids * 3, gy * 3):
        with torch.cuda.stream(s):
            got.append(grad(i, q))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want * 3))
    side = streams[0]
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        grad(ids[0], gy[0])
    torch.cuda.current_stream().wait_stream(side)
    graph, held = torch.cuda.CUDAGraph(), ids[0].clone()
    with torch.cuda.graph(graph):
        out = grad(held, gy[0])
    for _ in range(3):
        held.copy_(make_ids("padded", 5000, 700, g))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, grad(held.clone(), gy[0]))


@pytest.mark.parametrize("n,V", [(7, 33000), (300, 33000), (33000, 40)])
def test_offsets_past_32_bits(n, V):
    """A table, and gradient rows, of more than 2^31 elements. Whole numbers, whose sums are exact in fp32."""
    d, g = 65536, torch.Generator(device="cuda").manual_seed(12)
    W = torch.randint(-9, 10, (V, d), generator=g, device="cuda", dtype=torch.int8).bfloat16().requires_grad_()
    ids = torch.randint(0, V, (n,), generator=g, device="cuda")
    ids[0], ids[1], ids[-1] = V - 1, -1, V - 1
    y = embedding(ids, W)
    assert max(y.numel(), W.numel()) > 2 ** 31
    on = ids >= 0
    assert torch.equal(y[on], W.detach()[ids[on]]) and not y[1].any()
    gy = torch.randint(-9, 10, (n, d), generator=g, device="cuda", dtype=torch.int8).bfloat16()
    dW, = torch.autograd.grad(y, W, gy)
    want = torch.zeros(V, d, device="cuda").index_add_(0, ids[on], gy[on].float()).bfloat16()
    assert torch.equal(dW, want)
