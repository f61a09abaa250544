"""GreedyDecoder on 4-bit weights and under rules: the step on 4-bit weights against the fp32 step of a model that has the
weights they stand for, tokens under rules against the definition applied to the recorded logits, grammars as automata, and
what changes between generations."""
import copy

import pytest
import torch

from pragnosia_amd import fp4, rules
from pragnosia_amd._lib import PragnosiaError
from pragnosia_amd.decode import GreedyDecoder
from pragnosia_amd.model import LM
from pragnosia_amd.rules import TokenRules

pytestmark = pytest.mark.gpu
DEV = "cuda"


def model(mixer="aspin", d=256, vocab=500, layers=2, ctx=64, seed=0):
    torch.manual_seed(seed)
    m = LM(vocab=vocab, d=d, layers=layers, ctx=ctx, mixer=mixer).to(DEV).eval()
    with torch.no_grad():  # logits that spread, so that no two are nearly equal
        m.e.weight.mul_(8.0)
        for mx in m.mix:
            mx.gate.fill_(0.5)
    return m


def rounded(m, group):
    """The model with the weights that 4 bits stand for, wherever the decoder takes them so: the layers' own copies, the
    token table left as it is for the lookups (a head of its own)."""
    r = copy.deepcopy(m)
    q = lambda w: w.copy_(fp4.dequantize(fp4.quantize(w, group)))  # noqa: E731
    with torch.no_grad():
        for mx, mp in zip(r.mix, r.mlp):
            for lin in (mx.q, mx.k, mx.v, mx.wa, mp.a, mp.b):
                q(lin.weight)
            if mx.delta:
                q(mx.wb.weight)
            elif not mx.write_all:
                q(mx.wi.weight)
    return r


def prompt(B, P, vocab=500, seed=1):
    return torch.randint(0, vocab, (B, P), generator=torch.Generator().manual_seed(seed)).to(DEV)


@pytest.mark.parametrize("mixer,d", [("aspin", 256), ("dspin", 192), ("hspin", 256), ("hdspin", 256), ("hspin1", 256)])
@pytest.mark.parametrize("B", [1, 3, 6, 40])
def test_fp4_step_is_the_step_of_the_rounded_model(mixer, d, B):
    """Teacher-forced in effect: the same tokens come out, and the logits differ by fp32 rounding alone. The rounded model's
    head is given its own table, so its logits are taken from its hidden rows times that."""
    m = model(mixer, d)
    group = {1: 32, 3: 64, 6: 128, 40: 64}[B]
    x, n = prompt(B, 20), 24
    dec = GreedyDecoder(m, B, record_logits=True, weights="fp4", group=group)
    states, pw, lg = dec.prefill(x)
    dec.start(states, pw, lg, n)
    dec.replay(n)
    toks, got = dec.out[:n].t().clone(), dec.logits(n)
    # the same steps eagerly, from the same prefilled state, fed the same tokens
    r = rounded(m, group)
    head = fp4.dequantize(fp4.quantize(m.e.weight, group))
    states, pw, _ = dec.prefill(x)
    with torch.no_grad():
        for t in range(n - 1):
            h = m.e(toks[:, t:t + 1]) + m.p(torch.full((1,), pw, device=DEV, dtype=torch.long))
            for i, (mx, mp) in enumerate(zip(r.mix, r.mlp)):
                h, states[i] = mx(h, states[i])
                h = mp(h)
            want = torch.nn.functional.linear(r.n(h), head)[:, -1]
            pw = (pw + 1) % m.ctx
            off = ((got[:, t + 1] - want).abs().max() / want.abs().max()).item()
            assert off < 1e-4 * (t + 2), (t, off)  # (a carrier layer's step is held to 1e-4, and states carry it on)
            assert torch.equal(toks[:, t + 1], got[:, t + 1].argmax(-1))


def test_fp4_follows_the_parameters_and_restarts():
    m, x = model(), prompt(2, 10)
    dec = GreedyDecoder(m, 2, weights="fp4")
    a = dec.generate(x, 16)
    assert torch.equal(dec.generate(x, 16), a) and torch.equal(GreedyDecoder(m, 2, weights="fp4").generate(x, 16), a)
    with torch.no_grad():
        for p in m.parameters():
            p.add_(0.05 * torch.randn_like(p))
    b = dec.generate(x, 16)
    assert torch.equal(b, GreedyDecoder(m, 2, weights="fp4").generate(x, 16)) and not torch.equal(a, b)
    assert torch.equal(dec.generate(x, 40)[:, :16], b)  # (a longer run: captured again)


def test_refusals():
    m = model()
    for kw, what in ((dict(weights="int4"), "fp4"), (dict(weights="fp4", fused=False), "fused"),
                     (dict(weights="fp4", group=48), "group")):
        with pytest.raises((ValueError, PragnosiaError), match=what):
            GreedyDecoder(m, 1, **kw)
    with pytest.raises(PragnosiaError, match="repetition"):
        GreedyDecoder(m, 1, rules=TokenRules(repetition=0.0)).generate(prompt(1, 4), 8)
    bits = torch.zeros(3, 16, dtype=torch.int32, device=DEV)
    with pytest.raises(PragnosiaError, match="next"):
        GreedyDecoder(m, 1, rules=TokenRules(mask=bits, next=torch.zeros(2, 500, dtype=torch.int32,
                                                                          device=DEV))).generate(prompt(1, 4), 8)


def by_definition(dec, x, n, rule):
    """The tokens that the rule leaves of the recorded logits, one by one on the CPU in fp32."""
    lgs, toks = dec.logits(n).cpu(), dec.out[:n].t().cpu()
    B, V = toks.shape[0], lgs.shape[2]
    state = None if rule.next is None else (torch.zeros(B, dtype=torch.long) if rule.state is None else rule.state.cpu())
    of = lambda p, b: (p[b] if torch.is_tensor(p) else torch.tensor(float(p))).cpu()  # noqa: E731
    bad = []
    for b in range(B):
        said, s = [], None if state is None else int(state[b])
        for t in range(n):
            z = lgs[b, t].clone()
            words = torch.tensor(x[b].tolist() + said, dtype=torch.long)
            seen = torch.zeros(V, dtype=torch.bool)
            seen[words] = True
            times = torch.bincount(torch.tensor(said, dtype=torch.long), minlength=V)
            r = of(rule.repetition, b)
            z = torch.where(seen, torch.where(z > 0, z / r, z * r), z)
            z = torch.where(times > 0, z - of(rule.presence, b), z)
            z = torch.where(times > 0, z - of(rule.frequency, b) * times, z)
            if rule.bias is not None:
                ids, v = rule.bias[0].cpu(), rule.bias[1].cpu()
                ids, v = (ids, v) if ids.dim() == 1 else (ids[b], v[b])
                z[ids] += v
            if rule.mask is not None:
                line = s if s is not None else 0
                if 0 <= line < rule.mask.shape[0]:
                    bits = (rule.mask[line].cpu().long()[:, None] >> torch.arange(32) & 1).flatten()[:V]
                    z[bits == 0] = -torch.inf
                elif line >= rule.mask.shape[0]:
                    z[:] = -torch.inf
            want = -1 if z.max() == -torch.inf else int(z.argmax())
            got = int(toks[b, t])
            if got != want:
                bad.append((b, t, got, want))
            if got >= 0:
                said.append(got)
                if s is not None and 0 <= s < rule.next.shape[0]:
                    s = int(rule.next[s, got])
    return bad


def grammar(S, V, seed=0):
    """A random automaton: some words in each state, random successors, some of which end it."""
    g = torch.Generator().manual_seed(seed)
    allowed = torch.rand(S, V, generator=g) < 0.1
    bits = torch.zeros(S, (V + 31) // 32 * 32, dtype=torch.long)
    bits[:, :V] = allowed
    mask = (bits.view(S, -1, 32) << torch.arange(32)).sum(2).to(torch.int32).to(DEV)
    nxt = torch.randint(0, S, (S, V), generator=g).to(torch.int32)
    nxt[torch.rand(S, V, generator=g) < 0.05] = S
    nxt[torch.rand(S, V, generator=g) < 0.02] = -1
    return dict(mask=mask, next=nxt.to(DEV))


def kinds(B, V):
    g = torch.Generator().manual_seed(3)
    r = lambda *s: torch.rand(*s, generator=g).to(DEV)  # noqa: E731
    ids = torch.randperm(V, generator=g)[:30].to(DEV)
    return {"repetition": TokenRules(repetition=1.3),
            "all": TokenRules(1 + r(B), r(B), 0.5 * r(B), bias=(ids, 3 * r(30) - 1)),
            "static mask": TokenRules(mask=grammar(1, V)["mask"], presence=0.3),
            "grammar": TokenRules(frequency=0.2, **grammar(6, V), state=torch.arange(B, device=DEV) % 6)}


@pytest.mark.parametrize("kind", ["repetition", "all", "static mask", "grammar"])
@pytest.mark.parametrize("mixer,B,weights", [("aspin", 2, "fp4"), ("aspin", 1, None), ("dspin", 7, "fp4"),
                                             ("hspin", 6, None), ("fspin", 2, None)])
def test_tokens_under_rules(mixer, B, weights, kind):
    """Every path of a step (4-bit, fp32 by GEMV and by matrix cores, unfused) chooses what the rules leave."""
    m, x, n = model(mixer) if mixer != "fspin" else plain_model(), prompt(B, 12), 30
    rule = kinds(B, 500)[kind]
    dec = GreedyDecoder(m, B, record_logits=True, weights=weights, rules=rule)
    got = dec.generate(x, n)
    assert got.shape == (B, n) and not by_definition(dec, x, n, rule)
    if kind == "grammar":  # once nothing is left, nothing comes any more
        ended = (got == -1).cummax(1).values
        assert torch.equal(ended, got == -1)


def plain_model():
    torch.manual_seed(0)
    m = LM(vocab=500, d=128, layers=2, ctx=64, mixer="fspin").to(DEV).eval()
    with torch.no_grad():
        m.e.weight.mul_(8.0)
    return m


def test_rules_change_between_generations():
    """Values, shapes, the prompt's length and whether there are rules at all."""
    m, x = model(), prompt(2, 9)
    free = GreedyDecoder(m, 2).generate(x, 20)
    dec = GreedyDecoder(m, 2, record_logits=True)
    assert torch.equal(dec.generate(x, 20), free)
    for rule, p in ((TokenRules(repetition=1.5), x), (TokenRules(repetition=2.5), x), (kinds(2, 500)["all"], x),
                    (kinds(2, 500)["grammar"], prompt(2, 50)), (TokenRules(presence=1.0), x)):
        dec.rules = rule
        dec.generate(p, 20)
        assert not by_definition(dec, p, 20, rule)
    dec.rules = None
    assert torch.equal(dec.generate(x, 20), free)
    neutral = GreedyDecoder(m, 2, rules=TokenRules()).generate(x, 20)
    assert torch.equal(neutral, free)


def test_two_decoders_of_one_model():
    """Weights, histories and states are each decoder's own: replays that take turns give what each gives alone."""
    m, x = model(), prompt(2, 9)
    decs = [GreedyDecoder(m, 2, weights="fp4", rules=TokenRules(repetition=1.5)),
            GreedyDecoder(m, 2, weights="fp4", group=32, rules=kinds(2, 500)["grammar"]), GreedyDecoder(m, 2, weights="fp4")]
    want = [dec.generate(x, 33) for dec in decs]
    for dec in decs:
        states, pw, lg = dec.prefill(x)
        dec.start(states, pw, lg, 33, x)
    for _ in range(4):
        for dec in decs:
            dec.replay(9)
    for dec, w in zip(decs, want):
        assert torch.equal(dec.out[:33].t(), w)


def test_refused_rules_leave_the_decoder_as_it_was():
    m, x = plain_model(), prompt(2, 9)
    good = TokenRules(repetition=1.3)
    dec = GreedyDecoder(m, 2, rules=good)
    want = dec.generate(x, 20)
    rs, graph = dec.rs, dec.graph
    for bad in (TokenRules(next=torch.zeros(3, 500, dtype=torch.int32)), TokenRules(repetition=0.0),
                TokenRules(bias=(torch.zeros(3, dtype=torch.int64), torch.zeros(4)))):
        dec.rules = bad
        with pytest.raises(PragnosiaError):
            dec.generate(x, 20)
        assert dec.rs is rs and dec.graph is graph
    dec.rules = good
    assert torch.equal(dec.generate(x, 20), want) and dec.graph is graph
    dec.rules = None
    assert torch.equal(dec.generate(x, 20), GreedyDecoder(m, 2).generate(x, 20))


@pytest.mark.parametrize("B", [1, 5])
def test_advance(B):
    """History, lengths and states in place: room that ends, tokens and states outside their range, a strided history."""
    g = torch.Generator().manual_seed(B)
    S, V, L = 4, 37, 6
    wide = torch.randint(0, V, (B, L + 3), generator=g).to(DEV)
    history, before = wide[:, 1:1 + L], wide.clone()
    lengths = torch.tensor([0, L - 1, L, 3, -1][:B]).to(DEV)
    state = torch.tensor([1, -1, S, S - 1, 0][:B]).to(DEV)
    nxt = torch.randint(-1, S + 1, (S, V), generator=g).to(torch.int32).to(DEV)
    tokens = torch.tensor([5, 36, 7, -1, 9][:B]).to(DEV)
    was = lengths.clone(), state.clone()
    rules.advance(tokens, history, lengths, nxt, state)
    want = before.clone()
    for b in range(B):
        t, n, s = int(tokens[b]), int(was[0][b]), int(was[1][b])
        if t >= 0 and 0 <= n < L:
            want[b, 1 + n] = t
        assert int(lengths[b]) == (n + 1 if t >= 0 and 0 <= n < L else n)
        assert int(state[b]) == (int(nxt[s, t]) if t >= 0 and 0 <= s < S else s)
    assert torch.equal(wide, want)
    rules.advance(torch.full((B,), V, device=DEV), history, lengths, vocab=V)
    rules.advance(torch.full((B,), 1 << 40, device=DEV), next=nxt, state=state)
    assert torch.equal(wide, want)
