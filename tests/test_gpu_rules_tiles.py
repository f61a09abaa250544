"""Rules on logits where there are enough tiles for the largest, and tokens of several tiles in numbers of rows that do not
divide among the XCDs, against the definition in 64 bits over whole tensors."""
import math

import pytest
import torch

from pragnosia_amd import rules

pytestmark = pytest.mark.gpu
DEV = "cuda"
F32, BF16, F64 = torch.float32, torch.bfloat16, torch.float64


def inputs(B, V, L, M, S, dtype, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    r = lambda *s: torch.rand(*s, generator=g, device=DEV)  # noqa: E731
    i = lambda hi, *s: torch.randint(0, hi, s, generator=g, device=DEV)  # noqa: E731
    logits = (3 * torch.randn(B, V, generator=g, device=DEV)).to(dtype)
    history, lengths = i(V + 50, B, L) - 25, i(L + 1, B)  # (some ids outside the vocabulary)
    history[:, ::3] = history[:, :1]  # (some many times)
    ids = r(B, V).topk(M, 1).indices
    ids[r(B, M) < 0.2] = -1
    values = torch.where(r(B, M) < 0.2, -math.inf, 4 * torch.randn(B, M, generator=g, device=DEV))
    allowed = torch.zeros(S, (V + 31) // 32 * 32, dtype=torch.bool, device=DEV)
    allowed[:, :V] = r(S, V) < torch.where(r(S, 1) < 0.5, 0.9, 0.1)
    allowed[2] = False
    mask = (allowed.view(S, -1, 32).long() << torch.arange(32, device=DEV)).sum(2).to(torch.int32)
    state = i(S + 2, B) - 1
    state[:4] = torch.tensor([-1, S, 2, 0], device=DEV)
    kw = dict(history=history, lengths=lengths, prompt=(r(B) * (lengths + 1)).long(), repetition=1 + 0.5 * r(B), presence=r(B),
              frequency=0.3 * r(B), bias=(ids, values), mask=mask, state=state)
    return logits, kw, allowed[:, :V]


def by_definition(logits, kw, allowed):
    """(processed logits fp64, a bound of an fp32 computation's error: half a step of 2^-24 for each operation, doubled)."""
    x = logits.to(F64)
    B, V = x.shape
    h, at = kw["history"], torch.arange(kw["history"].shape[1], device=DEV)[None]
    there = (at < kw["lengths"][:, None]) & (h >= 0) & (h < V)
    count = lambda on: torch.zeros(B, V, device=DEV, dtype=F64).scatter_add_(1, h.clamp(0, V - 1), on.to(F64))  # noqa: E731
    seen, times = count(there) > 0, count(there & (at >= kw["prompt"][:, None]))
    p = {k: kw[k].to(F64)[:, None] for k in ("repetition", "presence", "frequency")}
    x = torch.where(seen, torch.where(x > 0, x / p["repetition"], x * p["repetition"]), x)
    bound = torch.where(seen, x.abs(), 0.0)
    x = torch.where(times > 0, x - p["presence"], x)
    bound = bound + torch.where(times > 0, x.abs() + (p["frequency"] * times).abs(), 0.0)
    x = x - p["frequency"] * times
    bound = bound + torch.where(times > 0, x.abs(), 0.0)
    ids, values = kw["bias"]
    add = torch.zeros(B, V + 1, device=DEV, dtype=F64).scatter_(1, torch.where(ids < 0, V, ids), values.to(F64))[:, :V]
    x = x + add
    bound = bound + torch.where((add != 0) & x.isfinite(), x.abs(), 0.0)
    s, S = kw["state"], allowed.shape[0]
    keep = allowed[s.clamp(0, S - 1)] & (s < S)[:, None] | (s < 0)[:, None]
    return torch.where(keep, x, -math.inf), 2.0 ** -23 * bound


def check(logits, kw, allowed):
    want, bound = by_definition(logits, kw, allowed)
    got = rules.apply_rules(logits, **kw)
    assert got.dtype == logits.dtype
    if logits.dtype == BF16:
        bound = bound * 1.01 + 2.0 ** -8 * want.abs()
    got = got.to(F64)
    assert ((got == want) | ((got - want).abs() <= bound)).all()
    del got, want, bound
    exact = rules.apply_rules(logits.float(), **kw)  # (fp32 throughout)
    top = exact.amax(1)
    token = rules.next_token(logits, **kw)
    assert torch.equal(token, torch.where(top == -math.inf, -1, exact.argmax(1)))
    assert token[1] == -1 and token[2] == -1 and token[0] >= 0
    return token


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("V", [40003, 40008])
@pytest.mark.parametrize("B", [176, 181])
def test_largest_tiles(B, V, dtype):
    """Three tiles of 16384 words to a row and 512 or more of them, for logits and for tokens."""
    check(*inputs(B, V, 300, 20, 6, dtype, B))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("B,V", [(67, 40003), (65, 131072), (64, 33000), (71, 32762), (9, 70001)])
def test_tokens_of_several_tiles(B, V, dtype):
    check(*inputs(B, V, 300, 20, 6, dtype, B))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_largest_tiles_under_long_lists(dtype):
    """More words of a tile than its list holds."""
    check(*inputs(176, 40003, 20000, 3000, 6, dtype, 1))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_largest_tiles_in_a_graph(dtype):
    logits, kw, _ = inputs(180, 40003, 300, 20, 6, dtype, 5)
    rules.next_token(logits, **kw), rules.apply_rules(logits, **kw)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        token, out = rules.next_token(logits, **kw), rules.apply_rules(logits, **kw)
    for n in (10, 300, 0, 77):
        kw["lengths"].fill_(n)
        logits.normal_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(token, rules.next_token(logits, **kw)) and torch.equal(out, rules.apply_rules(logits, **kw))
