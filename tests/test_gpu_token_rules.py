"""GreedyDecoder's rules beyond single generations: the states that a grammar begins in, what is refused, what is kept."""
import pytest
import torch

from pragnosia_amd import decode
from pragnosia_amd._lib import PragnosiaError
from pragnosia_amd.decode import GreedyDecoder
from pragnosia_amd.model import LM
from pragnosia_amd.rules import TokenRules

pytestmark = pytest.mark.gpu
DEV = "cuda"
V = 500


def model(mixer="aspin", d=256):
    torch.manual_seed(0)
    m = LM(vocab=V, d=d, layers=2, ctx=64, mixer=mixer).to(DEV).eval()
    with torch.no_grad():
        m.e.weight.mul_(8.0)
    return m


def prompt(B, P, seed=1):
    return torch.randint(0, V, (B, P), generator=torch.Generator().manual_seed(seed)).to(DEV)


def lines(S, share=0.1, seed=0, dev=DEV):
    """Words (S, V) that a grammar allows, and the same as bits."""
    allowed = torch.rand(S, V, generator=torch.Generator().manual_seed(seed)) < share
    bits = torch.zeros(S, (V + 31) // 32 * 32, dtype=torch.long)
    bits[:, :V] = allowed
    return allowed, (bits.view(S, -1, 32) << torch.arange(32)).sum(2).to(torch.int32).to(dev)


@pytest.mark.parametrize("mixer,d", [("aspin", 256), ("fspin", 128)])
@pytest.mark.parametrize("S", [1, 2, 3, 7])
def test_states_begin_at_zero_and_stay(S, mixer, d):
    """A mask without states or successors: every sequence is in state 0, however many lines there are."""
    B, n = 3, 20
    allowed, mask = lines(S)
    got = GreedyDecoder(model(mixer, d), B, rules=TokenRules(mask=mask)).generate(prompt(B, 9), n).cpu()
    assert (got >= 0).all() and allowed[0][got].all()
    first = GreedyDecoder(model(mixer, d), B, rules=TokenRules(mask=mask[:1])).generate(prompt(B, 9), n).cpu()
    assert torch.equal(got, first)
    # states of their own
    state = torch.arange(B, device=DEV) % S
    got = GreedyDecoder(model(mixer, d), B, rules=TokenRules(mask=mask, state=state)).generate(prompt(B, 9), n).cpu()
    assert all(allowed[b % S][got[b]].all() for b in range(B))


def refused():
    """Rules that differ from `TokenRules(repetition=1.3, mask=, next=)` in one thing a step does not take."""
    _, mask = lines(4, dev="cpu")
    nxt = torch.zeros(4, V, dtype=torch.int32)
    good = dict(repetition=9.0, mask=mask.roll(1, 0), next=nxt + 1)
    i = lambda *s: torch.zeros(*s, dtype=torch.long)  # noqa: E731
    return {"presence": good | dict(presence=float("inf")), "frequency": good | dict(frequency=1e39),
            "penalties' number": good | dict(frequency=torch.zeros(5)), "mask's width": dict(repetition=9.0, mask=mask[:, 1:]),
            "mask's type": good | dict(mask=mask.float()), "next's shape": good | dict(next=nxt[:, 1:]),
            "next's type": good | dict(next=nxt.float()), "next alone": dict(repetition=9.0, next=nxt),
            "state alone": dict(repetition=9.0, state=i(3)), "states' number": good | dict(state=i(5)),
            "state's type": good | dict(state=torch.zeros(3)), "list's ids": good | dict(bias=(torch.zeros(4), torch.zeros(4))),
            "list's rows": good | dict(bias=(i(2, 4), torch.zeros(2, 4))), "list's values": good | dict(bias=(i(4), torch.zeros(3))),
            "list of none": good | dict(bias=(torch.tensor(3), torch.tensor(1.0)))}


@pytest.mark.parametrize("what", list(refused()))
def test_refused_rules_write_nothing(what):
    """Nothing of the refused rules reaches the buffers: the run goes on as it would have."""
    B, n = 3, 33
    _, mask = lines(4)
    good = TokenRules(repetition=1.3, mask=mask, next=(torch.arange(4, device=DEV) + 1).remainder(4).int()[:, None].expand(4, V))
    x = prompt(B, 9)
    dec = GreedyDecoder(model(), B, rules=good)
    want = dec.generate(x, n)
    states, pw, lg = dec.prefill(x)
    dec.start(states, pw, lg, n, x)
    dec.replay(17)
    rs, graph = dec.rs, dec.graph
    buffers = [*rs.penalties, rs.mask, rs.next, rs.state, rs.history, rs.lengths, rs.prompt]
    before = [t.clone() for t in buffers]
    dec.rules = TokenRules(**refused()[what])
    with pytest.raises(PragnosiaError, match="TokenRules"):
        dec.generate(x, n)
    assert dec.rs is rs and dec.graph is graph and all(torch.equal(a, b) for a, b in zip(buffers, before))
    dec.replay(17)  # (the other half of the run)
    assert torch.equal(dec.out[:n].t(), want)


@pytest.mark.parametrize("x", [torch.zeros(2, 9, dtype=torch.long), torch.zeros(3, 9), torch.zeros(9, dtype=torch.long)])
def test_prompts_are_refused(x):
    """Of another number of sequences, of numbers that are no ids, of one dimension."""
    dec = GreedyDecoder(model(), 3, rules=TokenRules(repetition=1.3))
    states, pw, lg = dec.prefill(prompt(3, 9))
    with pytest.raises(PragnosiaError, match="prompt"):
        dec.start(states, pw, lg, 20, x.to(DEV))
    assert dec.rs is None and dec.graph is None


def test_one_value_for_every_sequence():
    """Penalties and states of one value, numbers of other types, successors in 64 bits, tensors on the CPU."""
    B, n, x = 3, 20, prompt(3, 9)
    _, mask = lines(4)
    nxt = torch.randint(0, 4, (4, V), generator=torch.Generator().manual_seed(5))
    ids = torch.arange(0, 60, 2)
    m = model()
    want = GreedyDecoder(m, B, rules=TokenRules(torch.full((B,), 1.5, device=DEV), 0.5, 1.0, (ids.to(DEV), ids.float().to(DEV)),
                                                mask, torch.full((B,), 2, device=DEV), nxt.int().to(DEV))).generate(x, n)
    got = GreedyDecoder(m, B, rules=TokenRules(torch.tensor(1.5).double(), torch.tensor([0.5]).half(), torch.tensor([1, 1, 1]),
                                               (ids.int(), ids), mask.long().cpu(), torch.tensor([2]), nxt)).generate(x, n)
    assert torch.equal(got, want)


def test_successors_past_32_bits():
    """A state of 2^40, as one of S, lets nothing follow; one of -2^40, as -1, anything."""
    B, n, x, (_, mask) = 2, 12, prompt(2, 9), lines(2)
    m = model()
    for far, near in ((1 << 40, 2), (1 << 32, 2), (-(1 << 40), -1)):
        runs = [GreedyDecoder(m, B, rules=TokenRules(mask=mask, next=torch.full((2, V), s, device=DEV))).generate(x, n)
                for s in (far, near)]
        assert torch.equal(*runs)
        assert (runs[0][:, 1:] == -1).all() == (far > 0)


@pytest.mark.parametrize("rules", [None, TokenRules(repetition=1.4)])
@pytest.mark.parametrize("mixer,d,weights", [("aspin", 256, None), ("aspin", 256, "fp4"), ("fspin", 128, None)])
def test_replays_past_the_end(mixer, d, weights, rules):
    """More steps than a run has room for: what was recorded of it stays, and the next run is as the first."""
    B, n, x = 2, 9, prompt(2, 12)
    dec = GreedyDecoder(model(mixer, d), B, record_logits=True, weights=weights, rules=rules)
    want = dec.generate(x, n)
    states, pw, lg = dec.prefill(x)
    dec.start(states, pw, lg, n, x)
    dec.replay(n)
    logits = dec.logits(n).clone()  # (of this run: the fp32 step adds with atomics, whose last bits differ by run)
    dec.replay(n)  # (the last rows that there are)
    out, lgs = dec.out.clone(), dec.lgs.clone()
    for _ in range(3):
        dec.replay(n)
    assert torch.equal(dec.out, out) and torch.equal(dec.lgs, lgs) and dec.out.shape == (n + 8, B)
    assert torch.equal(dec.out[:n].t(), want) and torch.equal(dec.logits(n), logits)
    assert torch.equal(dec.generate(x, n), want)


def test_a_capture_that_fails_leaves_no_graph(monkeypatch):
    """A graph whose buffers were let go cannot be replayed; the next start captures one."""
    x = prompt(2, 9)
    dec = GreedyDecoder(model(), 2, rules=TokenRules(repetition=1.3))
    want = dec.generate(x, 30)
    with monkeypatch.context() as patch:
        patch.setattr(dec, "_load_weights", lambda: (_ for _ in ()).throw(MemoryError("no room")))
        with pytest.raises(MemoryError):
            dec.generate(x, 60)
    assert dec.graph is None
    assert torch.equal(dec.generate(x, 60)[:, :30], want)


@pytest.mark.parametrize("rules", [None, TokenRules(repetition=1.4)])
@pytest.mark.parametrize("mixer", ["aspin", "dspin"])
def test_fp4_step_where_decode_gemm_covers_no_width(monkeypatch, mixer, rules):
    """The o-projection as a product of torch's, beside 4-bit weights: the logits of the step that covers it."""
    B, n, x, m = 6, 25, prompt(6, 12), model(mixer)
    runs = []
    for covered in (True, False):
        with monkeypatch.context() as patch:
            if not covered:
                patch.setattr(decode, "_gemm_layers_ok", lambda model: False)
            dec = GreedyDecoder(m, B, record_logits=True, weights="fp4", rules=rules)
            runs.append((dec.generate(x, n), dec.logits(n).clone()))
            assert dec.gemm is covered
    (want, a), (got, b) = runs
    assert torch.equal(got, want)
    for t in range(n):  # (a step is held to 1e-4, and states carry it on)
        assert (a[:, t] - b[:, t]).abs().max() <= 1e-4 * (t + 2) * a[:, t].abs().max()


@pytest.mark.parametrize("dtype", [torch.int8, torch.uint8, torch.int16, torch.int64])
def test_successors_of_other_integers(dtype):
    B, n, x, (_, mask) = 2, 12, prompt(2, 9), lines(4)
    nxt = torch.randint(0, 6, (4, V), generator=torch.Generator().manual_seed(6), dtype=torch.int32).to(DEV)
    m = model()
    want, got = (GreedyDecoder(m, B, rules=TokenRules(mask=mask, next=t)).generate(x, n) for t in (nxt, nxt.to(dtype)))
    assert torch.equal(got, want)
