"""GreedyDecoder's rules beyond single generations: the states that a grammar begins in, what is refused, what is kept."""
import pytest
import torch

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


def lines(S, share=0.1, seed=0):
    """Words (S, V) that a grammar allows, and the same as bits."""
    allowed = torch.rand(S, V, generator=torch.Generator().manual_seed(seed)) < share
    bits = torch.zeros(S, (V + 31) // 32 * 32, dtype=torch.long)
    bits[:, :V] = allowed
    return allowed, (bits.view(S, -1, 32) << torch.arange(32)).sum(2).to(torch.int32).to(DEV)


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
