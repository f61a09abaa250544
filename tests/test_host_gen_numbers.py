"""CPU checks of the rules' numbers: what fp32 does not hold is refused."""
import pytest
import torch

from pragnosia_amd import rules
from pragnosia_amd._lib import PragnosiaError


@pytest.mark.parametrize("name,p", [("repetition", 1e39), ("repetition", 1e-46), ("repetition", -1e39), ("presence", 1e39),
                                    ("presence", -1e39), ("frequency", 3.5e38), ("frequency", -float("inf"))])
def test_numbers_past_fp32_are_refused(monkeypatch, name, p):
    """Finite in 64 bits, but an infinity or zero where the kernels take them."""
    monkeypatch.setattr(rules, "_require_gpu", lambda *t: None)
    monkeypatch.setattr(rules, "gen_lib", lambda: pytest.fail("the call reached the C ABI"))
    for call in (rules.next_token, rules.apply_rules):
        with pytest.raises(PragnosiaError, match=f"{name} must be finite"):
            call(torch.zeros(2, 10), **{name: p})


@pytest.mark.parametrize("kw", [dict(repetition=2.0 ** -149), dict(repetition=torch.finfo(torch.float32).max),
                                dict(presence=torch.finfo(torch.float32).max), dict(presence=3, frequency=-2, repetition=2)])
def test_numbers_within_fp32_are_taken(monkeypatch, kw):
    made = []
    monkeypatch.setattr(rules, "_require_gpu", lambda *t: None)
    monkeypatch.setattr(rules, "_call", lambda what, *args: made.append(what))
    rules.apply_rules(torch.zeros(2, 10), **kw)
    assert made == ["pragnosia_rules"]


@pytest.mark.gpu
@pytest.mark.parametrize("kw", [dict(repetition=1e39), dict(repetition=1e-46), dict(presence=1e39), dict(frequency=-1e39)])
def test_numbers_past_fp32_on_the_gpu(kw):
    """By the short way too, which looks for itself."""
    for call in (rules.next_token, rules.apply_rules):
        with pytest.raises(PragnosiaError, match="must be finite"):
            call(torch.zeros(2, 10, device="cuda"), **kw)
