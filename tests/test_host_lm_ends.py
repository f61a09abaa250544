"""CPU checks of the language model's two ends: the second header's exports, binding and version, what the entry points
and the Python functions refuse before anything is launched, and the workspace queries."""
import ctypes
import os
import re

import pytest
import torch

from pragnosia_amd import embed, head
from pragnosia_amd._lib import LM_SIGNATURES, PragnosiaError, lm_lib

HEADER = os.path.join(os.path.dirname(os.path.abspath(head.__file__)), "include", "pragnosia_lm.h")
null, one, odd = ctypes.c_void_p(0), ctypes.c_void_p(16), ctypes.c_void_p(24)


@pytest.fixture(scope="module")
def L():
    return lm_lib()


def test_header_exports_and_binding(L):
    txt = re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S)
    names = re.findall(r"^\s*\w+\s*\**\s*(pragnosia_\w+)\s*\(", txt, flags=re.M)
    assert set(names) == set(LM_SIGNATURES) and len(names) == 8
    for n in names:
        assert hasattr(L, n)
        args = re.search(n + r"\s*\((.*?)\)", txt, flags=re.S).group(1)
        count = 0 if args.strip() == "void" else args.count(",") + 1
        assert len(LM_SIGNATURES[n]) == count, n
    assert f"ABI version of this header ({L.pragnosia_lm_abi_version()})" in open(HEADER).read()


def fwd(L, n=4, V=10, d=16, K=0, h=one, W=one, y=one, ids=null, z=null, tau=1.0, out=one, kd=null, ws=one,
        size=1 << 30):
    return L.pragnosia_head_fwd(h, W, y, ids, z, tau, out, out, kd, kd, kd, kd, kd, kd, ws, size, n, V, d, K, null)


@pytest.mark.parametrize("bad", [dict(n=0), dict(n=-1), dict(V=0), dict(d=12), dict(d=0), dict(K=-1), dict(h=null),
                                 dict(h=odd), dict(W=odd), dict(out=null), dict(y=null), dict(tau=0.0),
                                 dict(tau=float("nan")), dict(tau=float("inf")), dict(tau=2.0 ** -11),
                                 dict(tau=2.0 ** 11), dict(ids=one), dict(K=3),
                                 dict(K=3, ids=one, z=one), dict(K=1025, ids=one, z=one, kd=one), dict(ws=null),
                                 dict(ws=odd), dict(size=16), dict(n=1 << 25), dict(V=1 << 25)])
def test_forward_refuses(L, bad):
    assert fwd(L, **bad) == -1


def bwd(L, n=4, V=10, d=16, K=0, g=one, gk=null, y=one, lse=one, kd=null, tau=1.0, dh=one, dW=one, ws=one,
        size=1 << 30):
    return L.pragnosia_head_bwd(g, null, gk, one, one, y, lse, kd, kd, kd, kd, kd, tau, dh, dW, 0, ws, size, n, V, d, K,
                                null)


@pytest.mark.parametrize("bad", [dict(n=0), dict(d=4), dict(g=null), dict(g=odd), dict(y=null), dict(lse=null),
                                 dict(gk=one), dict(gk=one, K=2), dict(gk=one, kd=one), dict(dh=null, dW=null),
                                 dict(dW=odd), dict(tau=-1.0), dict(ws=null), dict(size=64)])
def test_backward_refuses(L, bad):
    assert bwd(L, **bad) == -1


def test_embed_refuses(L):
    f = lambda n=4, V=10, d=8, W=one, ids=one, y=one: L.pragnosia_embed_fwd(ids, W, 0, 1.0, y, 0, null, n, V, d, null)
    for bad in (dict(n=-1), dict(V=0), dict(d=12), dict(d=0), dict(W=null), dict(W=odd), dict(ids=null), dict(y=odd),
                dict(V=1 << 30)):
        assert f(**bad) == -1, bad
    assert f(n=0, ids=null, y=null) == 0  # nothing to do
    b = lambda n=4, V=10, d=8, g=one, k=one, dW=one, ws=one, size=1 << 30: L.pragnosia_embed_bwd(
        g, 0, k, 1, 1.0, dW, 0, ws, size, n, V, d, null)
    for bad in (dict(n=-1), dict(d=4), dict(g=null), dict(g=odd), dict(k=null), dict(dW=null), dict(n=300, ws=null),
                dict(n=300, size=64)):
        assert b(**bad) == -1, bad


def test_workspace_queries(L):
    assert L.pragnosia_head_fwd_workspace_bytes(0, 8, 8, 0) == -1
    assert L.pragnosia_head_bwd_workspace_bytes(8, 8, 9) == -1
    assert L.pragnosia_embed_bwd_workspace_bytes(8, 0, 8) == -1
    assert L.pragnosia_embed_bwd_workspace_bytes(256, 8, 8) == 0 < L.pragnosia_embed_bwd_workspace_bytes(257, 8, 8)
    # the backward's space stays near its limit whatever the vocabulary, and grows with the tokens by what they need
    for n, V, d in ((16384, 32768, 768), (8192, 262144, 1024), (100, 1 << 20, 512), (1, 1, 8)):
        assert 0 < L.pragnosia_head_bwd_workspace_bytes(n, V, d) < (512 << 20) + 16 * n * d
    assert L.pragnosia_head_bwd_workspace_bytes(8192, 8192, 768) < 160 << 20
    with pytest.raises(PragnosiaError, match="rejected"):
        head._workspace("pragnosia_head_bwd_workspace_bytes", 8, 8, 9)


def test_no_cpu_path():
    h, W, y = torch.zeros(3, 16), torch.zeros(5, 16), torch.zeros(3, dtype=torch.long)
    with pytest.raises(PragnosiaError, match="no CPU fallback"):
        head.linear_cross_entropy(h, W, y)
    with pytest.raises(PragnosiaError, match="no CPU fallback"):
        head.linear_distill(h, W, torch.zeros(3, 2, dtype=torch.long), torch.zeros(3, 2))
    with pytest.raises(PragnosiaError, match="no CPU fallback"):
        embed.embedding(y, W)


@pytest.fixture
def unguarded(monkeypatch):
    """The calls below carry a mismatch each, so none gets as far as a launch."""
    for mod in (head, embed):
        monkeypatch.setattr(mod, "_require_gpu", lambda *t: None)
        monkeypatch.setattr(mod, "lm_lib", lambda: pytest.fail("a mismatched call reached the C ABI"))


z = torch.zeros
L64 = dict(dtype=torch.long)


@pytest.mark.parametrize("h,W,y,what", [
    (z(3, 16), z(5, 24), z(3, **L64), "W has shape"), (z(3, 16), z(5, 16), z(4, **L64), "leading sizes"),
    (z(3, 12), z(5, 12), z(3, **L64), "multiple of 8"), (z(3, 16), z(0, 16), z(3, **L64), "not empty"),
    (z(3, 16), z(5, 16), z(3), "integers"), (z(3, 16).half(), z(5, 16), z(3, **L64), "bf16 or fp32"),
    (z(3, 16), z(5, 16).double(), z(3, **L64), "bf16 or fp32"),
    (z(2, 3, 16), z(5, 16), z(3, 2, **L64), "leading sizes"),
    (z(3, 16), z(5), z(3, **L64), "expected")])
def test_cross_entropy_refuses(unguarded, h, W, y, what):
    with pytest.raises(PragnosiaError, match=what):
        head.linear_cross_entropy(h, W, y)


@pytest.mark.parametrize("ids,lg,tau,what", [
    (z(3, 2, **L64), z(3, 3), 1.0, "logits has shape"), (z(4, 2, **L64), z(4, 2), 1.0, "leading sizes"),
    (z(3, 0, **L64), z(3, 0), 1.0, "K from 1"), (z(3, 1025, **L64), z(3, 1025), 1.0, "K from 1"),
    (z(3, 2), z(3, 2), 1.0, "integers"), (z(3, 2, **L64), z(3, 2, **L64), 1.0, "floating"),
    (z(3, 2, **L64), z(3, 2), 0.0, "tau"), (z(3, 2, **L64), z(3, 2), float("nan"), "tau"),
    (z(3, 2, **L64), z(3, 2), 2.0 ** -11, "tau"), (z(3, 2, **L64), z(3, 2), 1e30, "tau"),
    (z(3, **L64), z(3, 2), 1.0, "leading sizes")])
def test_distill_refuses(unguarded, ids, lg, tau, what):
    with pytest.raises(PragnosiaError, match=what):
        head.linear_distill(z(3, 16), z(5, 16), ids, lg, tau)


@pytest.mark.parametrize("ids,W,kw,what", [
    (z(3), z(5, 16), {}, "integers"), (z(3, **L64), z(5, 12), {}, "multiple of 8"),
    (z(3, **L64), z(0, 16), {}, "V > 0"), (z(3, **L64), z(5, 16).half(), {}, "bf16 or fp32"),
    (z(3, **L64), z(5, 16), dict(dtype=torch.float64), "bf16 or fp32"),
    (z(3, **L64), z(5, 16), dict(scale=float("inf")), "finite"), (z(3, **L64), z(5, 4, 4), {}, "W has shape")])
def test_embedding_refuses(unguarded, ids, W, kw, what):
    with pytest.raises(PragnosiaError, match=what):
        embed.embedding(ids, W, **kw)


def test_fused_model_on_the_cpu():
    """The parameters, names and initial draw are the plain model's; on the CPU the lookups and the loss are torch's."""
    from pragnosia_amd.model import LM
    a, b = (torch.manual_seed(0) and LM(vocab=40, d=64, layers=1, ctx=16, fused_ends=f) for f in (False, True))
    assert list(a.state_dict()) == list(b.state_dict())
    assert all(torch.equal(p, q) for p, q in zip(a.parameters(), b.parameters()))
    x = torch.randint(0, 40, (2, 16))
    assert torch.equal(a.e(x), b.e(x))
    h = torch.randn(2, 16, 64)
    assert torch.equal(a.loss(h, x), b.loss(h, x))
