"""Arguments without dimensions, or with empty ones, are refused as others of a wrong shape are."""
import pytest
import torch

from pragnosia_amd import fp4, rules
from pragnosia_amd._lib import PragnosiaError

z, L64 = torch.zeros, dict(dtype=torch.long)


@pytest.fixture
def unguarded(monkeypatch):
    for mod in (fp4, rules):
        monkeypatch.setattr(mod, "_require_gpu", lambda *t: None)
        monkeypatch.setattr(mod, "gen_lib", lambda: pytest.fail("a mismatched call reached the C ABI"))


@pytest.mark.parametrize("x", [z(2, 3, 0), z(2, 0), z(0), z(0, 3, 0)])
def test_rows_of_no_columns(unguarded, x):
    nbytes, count = fp4._sizes("", 16, 64, 32)
    Q = fp4.Weight4(z(nbytes, dtype=torch.uint8), z(count, dtype=torch.bfloat16), 16, 64, 32)
    with pytest.raises(PragnosiaError, match="x \\(..., 64\\)"):
        fp4.linear(x, Q)


@pytest.mark.parametrize("next", [z((), dtype=torch.int32), z(10, dtype=torch.int32), z(3, 0, dtype=torch.int32)])
def test_successors_without_states(unguarded, next):
    with pytest.raises(PragnosiaError, match="next"):
        rules.advance(z(2, **L64), next=next, state=z(2, **L64))


@pytest.mark.parametrize("kw", [dict(bias=(z((), **L64), z(()))), dict(mask=z((), dtype=torch.int32)),
                                dict(history=z((), **L64)), dict(repetition=z(())), dict(bias=(z(3, **L64), z(())))])
@pytest.mark.parametrize("dev", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_rules_without_dimensions(monkeypatch, kw, dev):
    f = lambda v: tuple(map(f, v)) if isinstance(v, tuple) else v.to(dev)  # noqa: E731
    monkeypatch.setattr(rules, "_require_gpu", lambda *t: None)
    for call in (rules.next_token, rules.apply_rules):
        with pytest.raises(PragnosiaError, match="bias|mask|history|repetition"):
            call(z(2, 10, device=dev), **{k: f(v) for k, v in kw.items()})
