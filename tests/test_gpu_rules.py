"""Rules on logits against the definition in 64 bits, word by word on the CPU: penalties, biases, masks, the token they
leave; odd vocabularies and alignments, empty histories and masks, ids outside the vocabulary."""
import math

import pytest
import torch

from pragnosia_amd import rules
from pragnosia_amd._lib import PragnosiaError

pytestmark = pytest.mark.gpu
DEV = "cuda"
F32, BF16 = torch.float32, torch.bfloat16


def inputs(B, V, L, M=0, S=0, dtype=F32, seed=0):
    """A call's arguments on the CPU."""
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.rand(*s, generator=g)  # noqa: E731
    lengths = torch.randint(0, L + 1, (B,), generator=g) if L else None
    if L:
        lengths[0] = L
    kw = dict(logits=(3 * torch.randn(B, V, generator=g)).to(dtype), repetition=1 + 0.5 * r(B), presence=r(B),
              frequency=0.3 * r(B))
    if L:
        kw |= dict(history=torch.randint(0, max(2, V // 3), (B, L), generator=g), lengths=lengths,
                   prompt=(r(B) * (lengths + 1)).long())
    if M:
        ids = torch.stack([torch.randperm(V, generator=g)[:M] for _ in range(B)])
        ids[r(B, ids.shape[1]) < 0.2] = -1
        kw |= dict(bias=(ids, torch.where(r(*ids.shape) < 0.2, -math.inf, 4 * torch.randn(ids.shape, generator=g))))
    if S:
        allowed = r(S, V) < torch.where(r(S, 1) < 0.5, 0.9, 0.1)
        if S > 2:
            allowed[2] = False
        kw |= dict(mask=pack(allowed), state=torch.randint(-1, S + 2, (B,), generator=g))
        if S > 2:
            kw["state"][-1] = 2
    return kw


def pack(allowed):
    """Truth values (S, V) as bits."""
    S, V = allowed.shape
    bits = torch.zeros(S, (V + 31) // 32 * 32, dtype=torch.long)
    bits[:, :V] = allowed
    return (bits.view(S, -1, 32) << torch.arange(32)).sum(2).to(torch.int32)


def gpu(kw):
    f = lambda v: tuple(map(f, v)) if isinstance(v, tuple) else v.to(DEV) if torch.is_tensor(v) else v  # noqa: E731
    kw = {k: f(v) for k, v in kw.items()}
    return kw.pop("logits"), kw


def by_definition(logits, history=None, lengths=None, prompt=None, repetition=1.0, presence=0.0, frequency=0.0, bias=None,
                  mask=None, state=None):
    """(processed logits fp64, a bound of an fp32 computation's error)."""
    x = logits.double().clone()
    B, V = x.shape
    of = lambda p, b: float(p[b]) if torch.is_tensor(p) else p  # noqa: E731
    bound = torch.zeros(B, V, dtype=torch.float64)
    for b in range(B):
        L = 0 if history is None else history.shape[1]
        n = L if lengths is None else min(max(int(lengths[b]), 0), L)
        start = 0 if prompt is None else min(max(int(prompt[b]), 0), n)
        seen, times = set(), {}
        for t in range(n):
            v = int(history[b, t])
            if 0 <= v < V:
                seen.add(v)
                if t >= start:
                    times[v] = times.get(v, 0) + 1
        r = of(repetition, b)
        for v in seen:
            steps = [abs(float(x[b, v]))]
            x[b, v] = x[b, v] / r if x[b, v] > 0 else x[b, v] * r
            steps.append(abs(float(x[b, v])))
            if v in times:
                x[b, v] -= of(presence, b)
                steps.append(abs(float(x[b, v])))
                x[b, v] -= of(frequency, b) * times[v]
                steps += [abs(float(x[b, v])), abs(of(frequency, b) * times[v])]
            bound[b, v] = 2.0 ** -24 * sum(s for s in steps[1:] if math.isfinite(s))
        if bias is not None:
            ids, values = (t if t.dim() == 1 else t[b] for t in bias)
            last = {int(i): float(v) for i, v in zip(ids, values)}
            for v, value in last.items():
                if 0 <= v < V:
                    x[b, v] += value
                    if math.isfinite(float(x[b, v])):
                        bound[b, v] += 2.0 ** -24 * abs(float(x[b, v]))
        if mask is not None:
            S = mask.shape[0]
            line = int(state[b]) if state is not None else 0 if S == 1 else b
            if line >= S:
                x[b] = -math.inf
            elif line >= 0:
                bits = (mask[line].long()[:, None] >> torch.arange(32) & 1).flatten()[:V]
                x[b, bits == 0] = -math.inf
    return x, 2 * bound


def check(kw):
    """Both functions; the token is checked against the processed fp32 values where these are bf16's whole ones."""
    want, bound = by_definition(**kw)
    logits, args = gpu(kw)
    got = rules.apply_rules(logits, **args)
    assert got.dtype == logits.dtype and got.shape == logits.shape
    got = got.double().cpu()
    if logits.dtype == BF16:
        bound = bound * 1.01 + 2.0 ** -8 * want.abs()
    same = (got == want) | (got.isnan() & want.isnan())
    assert (same | ((got - want).abs() <= bound)).all()
    token = rules.next_token(logits, **args).cpu()
    assert token.dtype == torch.int64
    exact = rules.apply_rules(logits.float(), **args).cpu()  # (fp32 throughout)
    top = exact.amax(1)
    assert torch.equal(token, torch.where(top == -math.inf, -1, exact.argmax(1)))
    return token


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("V", [1, 7, 32, 33, 501, 4093, 8192, 8200, 16381, 40003])
def test_vocabularies(V, dtype):
    """One to several tiles, rows that start anywhere in a vector, everything at once."""
    check(inputs(5, V, 60, M=min(V, 20), S=4, dtype=dtype, seed=V))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("L", [0, 1, 2, 1023, 1024, 1025, 9000])
def test_histories(L, dtype):
    check(inputs(3, 1000, L, dtype=dtype, seed=L))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("V,L,M", [(40000, 20000, 0), (9000, 6000, 5000)])
def test_many_words_repeated(V, L, M, dtype):
    """More words of one tile under rules than its list of them holds."""
    check(inputs(2, V, L, M=M, S=2, dtype=dtype, seed=7))


@pytest.mark.parametrize("M", [1, 300, 2500])
def test_lists(M):
    check(inputs(2, 3001, 5, M=M, seed=M))


@pytest.mark.parametrize("S", [1, 2, 50])
def test_masks(S):
    kw = inputs(6, 20000, 30, S=S, seed=S)
    check(kw)
    for drop in (0, 1):  # without states: line by row, or the only one
        kw.pop("state", None)
        kw["mask"] = pack(torch.rand(6 if drop else 1, 20000, generator=torch.Generator().manual_seed(S)) < 0.3)
        check(kw)


def test_many_rows():
    """Enough tiles that the largest are taken (fp32), and a batch of them."""
    check(inputs(40, 33000, 20, M=3, S=5, seed=3))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("B", [7, 8, 24, 63, 64, 67])
def test_many_rows_of_several_tiles(B, dtype):
    check(inputs(B, 17000 if B > 8 else 35001, 40, M=3, S=5, dtype=dtype, seed=B))


def test_nothing_left():
    kw = inputs(4, 9000, 10, S=3, seed=9)
    kw["state"] = torch.tensor([0, 2, 3, 1 << 40])
    assert (check(kw)[1:] == -1).all()
    x = torch.full((2, 50), -math.inf)
    assert check(dict(logits=x)).tolist() == [-1, -1]
    x[1, 49] = torch.finfo(F32).min
    assert check(dict(logits=x)).tolist() == [-1, 49]
    ids = torch.arange(50)
    assert check(dict(logits=torch.zeros(2, 50), bias=(ids, torch.full((50,), -math.inf)))).tolist() == [-1, -1]


def test_ties_and_special_values():
    x = torch.zeros(6, 700)
    x[0, [5, 600]] = 2.0
    x[1, 3], x[1, 650] = -0.0, 0.0       # equal: the lowest of all
    x[2, 9], x[2, 400] = math.nan, math.inf
    x[3] = -math.inf
    x[3, 77] = torch.finfo(F32).min
    x[4] = torch.finfo(F32).min
    x[5, 1] = -math.nan
    assert check(dict(logits=x)).tolist() == [5, 0, 9, 77, 0, 1]
    # a masked NaN or infinity is no candidate
    allowed = torch.ones(1, 700, dtype=torch.bool)
    allowed[0, [9, 400, 5, 1]] = False
    assert check(dict(logits=x, mask=pack(allowed))).tolist() == [600, 0, 0, 77, 0, 0]
    # infinities under penalties and biases
    x = torch.tensor([[math.inf, -math.inf, 1.0, 0.0]])
    check(dict(logits=x, history=torch.tensor([[0, 1, 2, 3]]), repetition=2.0, presence=0.5,
               bias=(torch.tensor([0, 1]), torch.tensor([-math.inf, 3.0]))))


def test_numbers_shared_lists_and_ids_outside():
    """Penalties as numbers, a list for all rows, ids outside the vocabulary, repeated entries (the last counts), lengths
    and prompts outside the history."""
    g = torch.Generator().manual_seed(5)
    h = torch.randint(-3, 130, (4, 64), generator=g)
    h[0, :5] = torch.tensor([-1, 100, 1 << 40, -(1 << 40), 99])
    ids = torch.tensor([3, 7, 3, -1, 100, 1 << 35, 99, 3])
    kw = dict(logits=torch.randn(4, 100, generator=g), history=h, lengths=torch.tensor([-4, 64, 1 << 40, 30]),
              prompt=torch.tensor([-1, 1 << 40, -(1 << 40), 12]), repetition=1.7, presence=0.25, frequency=0.5,
              bias=(ids, torch.arange(8.0)))
    check(kw)
    kw.pop("lengths"), kw.pop("prompt")
    check(kw)
    check(dict(logits=kw["logits"], history=h[:, :0], bias=(ids[:0], torch.zeros(0))))
    check(dict(logits=kw["logits"], history=h.to(torch.int32).clamp(-2, 120), repetition=0.5))


def test_integer_types_views_and_rows():
    logits, kw = gpu(inputs(3, 777, 40, M=8, S=3, seed=2))
    want, best = rules.apply_rules(logits, **kw), rules.next_token(logits, **kw)
    wide = torch.zeros(3, 100, dtype=torch.long, device=DEV)
    wide[:, 13:53] = kw["history"]
    args = kw | dict(history=wide[:, 13:53], lengths=kw["lengths"].int(), prompt=kw["prompt"].int(),
                     state=kw["state"].int(), bias=(kw["bias"][0].int(), kw["bias"][1].double()))
    big = torch.zeros(3, 900, device=DEV)
    big[:, 5:782] = logits
    assert torch.equal(rules.apply_rules(big[:, 5:782], **args), want)
    assert torch.equal(rules.next_token(big[:, 5:782], **args), best)
    each = [rules.next_token(logits[b:b + 1], kw["history"][b:b + 1], kw["lengths"][b:b + 1], kw["prompt"][b:b + 1],
                             repetition=kw["repetition"][b:b + 1], presence=kw["presence"][b:b + 1],
                             frequency=kw["frequency"][b:b + 1], bias=tuple(t[b:b + 1] for t in kw["bias"]),
                             mask=kw["mask"], state=kw["state"][b:b + 1]) for b in range(3)]
    assert torch.equal(torch.cat(each), best)
    assert rules.next_token(logits[:0]).shape == (0,) and rules.apply_rules(logits[:0]).shape == (0, 777)


def test_graph_and_streams():
    """Captured: the history grows on the device between replays."""
    B, V = 3, 20011
    logits, kw = gpu(inputs(B, V, 50, M=5, S=4, seed=4))
    kw["lengths"] = torch.full((B,), 10, device=DEV)
    kw["prompt"] = torch.full((B,), 4, device=DEV)
    rules.next_token(logits, **kw)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        token, out = rules.next_token(logits, **kw), rules.apply_rules(logits, **kw)
    for n in (10, 25, 50, 0):
        kw["lengths"].fill_(n)
        logits.normal_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(token, rules.next_token(logits, **kw)) and torch.equal(out, rules.apply_rules(logits, **kw))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = rules.next_token(logits, **kw)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(other, rules.next_token(logits, **kw))


def test_two_graphs_at_once():
    """Rows of several tiles, whose best words pass through a workspace: two captured calls replayed on two streams, and
    eager ones between."""
    calls = []
    for seed in (1, 2):
        logits, kw = gpu(inputs(16, 70001, 40, M=3, S=4, seed=seed))
        want = rules.next_token(logits, **kw)
        g, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        with torch.cuda.graph(g):
            token = rules.next_token(logits, **kw)
        calls.append((g, stream, token, want, logits, kw))
    for _ in range(10):
        for g, stream, token, *_ in calls:
            stream.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(stream):
                token.zero_()
                for _ in range(5):
                    g.replay()
        eager = [rules.next_token(logits, **kw) for *_, logits, kw in calls]
        torch.cuda.synchronize()
        for (_, _, token, want, _, _), got in zip(calls, eager):
            assert torch.equal(token, want) and torch.equal(got, want)


def test_trace():
    from torch.fx.experimental.proxy_tensor import make_fx
    logits, kw = gpu(inputs(2, 100, 8, M=3, S=2, seed=6))
    f = lambda x: rules.next_token(x, **kw)  # noqa: E731
    traced = make_fx(f)(logits)
    assert "rules_token" in traced.code and torch.equal(traced(logits), f(logits))
    f = lambda x: rules.apply_rules(x, kw["history"], repetition=1.5, presence=kw["presence"])  # noqa: E731
    traced = make_fx(f)(logits)
    assert "rules_apply" in traced.code and torch.equal(traced(logits), f(logits))


def test_refuses_gradients():
    x = torch.zeros(2, 10, device=DEV, requires_grad=True)
    with pytest.raises(PragnosiaError, match="no backward"):
        rules.next_token(x)


def test_large_offsets():
    """Logits past 2^31 elements, the best word in the last row's last place."""
    B, V = 600, 4_000_003
    x = torch.zeros(B, V, device=DEV, dtype=BF16)
    x[-1, -1], x[B // 2, 5], x[0, V - 2] = 3.0, 2.0, 1.0
    got = rules.next_token(x, history=torch.full((B, 1), V - 1, device=DEV), repetition=2.0)
    assert got[-1] == V - 1 and got[B // 2] == 5 and got[0] == V - 2 and got[1] == 0
    out = rules.apply_rules(x, history=torch.full((B, 1), V - 1, device=DEV), repetition=2.0)
    assert out[-1, -1] == 1.5 and out[B // 2, 5] == 2 and out[:, 6:100].count_nonzero() == 0
