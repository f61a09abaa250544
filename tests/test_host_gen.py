"""CPU checks of generation's operators: the third header's exports, binding and version, what the entry points and the
Python functions refuse before anything is launched, and the size queries."""
import copy
import ctypes
import os
import pickle
import re

import pytest
import torch

from pragnosia_amd import fp4, rules
from pragnosia_amd._lib import GEN_SIGNATURES, PragnosiaError, gen_lib

HEADER = os.path.join(os.path.dirname(os.path.abspath(fp4.__file__)), "include", "pragnosia_gen.h")
null, one, odd, far = (ctypes.c_void_p(v) for v in (0, 16, 24, 1 << 44))
z = torch.zeros
L64 = dict(dtype=torch.long)


@pytest.fixture(scope="module")
def L():
    return gen_lib()


def test_header_exports_and_binding(L):
    txt = re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S)
    names = re.findall(r"^\s*\w+\s*\**\s*(pragnosia_\w+)\s*\(", txt, flags=re.M)
    assert set(names) == set(GEN_SIGNATURES)
    for n in names:
        assert hasattr(L, n)
        args = re.search(n + r"\s*\((.*?)\)", txt, flags=re.S).group(1)
        count = 0 if args.strip() == "void" else args.count(",") + 1
        assert len(GEN_SIGNATURES[n]) == count, n
    assert f"ABI version of this header ({L.pragnosia_gen_abi_version()})" in open(HEADER).read()


def test_sizes(L):
    assert L.pragnosia_fp4_code_bytes(1, 8) == 1024 and L.pragnosia_fp4_code_bytes(17, 136) == 4096
    assert L.pragnosia_fp4_scale_bytes(17, 136, 32) == 512 and L.pragnosia_fp4_scale_bytes(16, 128, 128) == 32
    for N, K, g in ((0, 8, 32), (1, 0, 32), (1, 12, 32), (1, 65544, 32), ((1 << 26) + 1, 8, 32)):
        assert L.pragnosia_fp4_code_bytes(N, K) == -1 and L.pragnosia_fp4_scale_bytes(N, K, g) == -1
    assert L.pragnosia_fp4_scale_bytes(16, 128, 16) == -1
    assert fp4._sizes("", 1000, 1000, 64) == (L.pragnosia_fp4_code_bytes(1000, 1000),
                                              L.pragnosia_fp4_scale_bytes(1000, 1000, 64) // 2)
    # of tokens alone, and only where a row has several tiles
    assert L.pragnosia_rules_workspace_bytes(4, 32761) == 0 < L.pragnosia_rules_workspace_bytes(4, 32762)
    assert L.pragnosia_rules_workspace_bytes(0, 9) == 0
    for B, V in ((-1, 9), (65536, 9), (1, 0), (1, (1 << 26) + 1), (65535, 1 << 26)):
        assert L.pragnosia_rules_workspace_bytes(B, V) == -1


def linear(L, x=one, codes=one, scales=one, lnw=null, lnb=null, eps=1e-5, bias=null, act=0, resid=null, y=far, n=4, N=16,
           K=64, group=32, bf16=0):
    return L.pragnosia_fp4_linear(x, bf16, codes, scales, lnw, lnb, eps, bias, act, resid, y, n, N, K, group, null)


@pytest.mark.parametrize("bad", [
    dict(x=null), dict(x=odd), dict(codes=null), dict(codes=odd), dict(scales=odd), dict(y=null), dict(lnb=one),
    dict(lnw=odd), dict(lnw=one, eps=-1.0), dict(lnw=one, eps=float("nan")), dict(act=2), dict(n=-1), dict(n=1 << 25),
    dict(n=1 << 24, N=128), dict(n=1 << 24, K=128), dict(N=0), dict(K=60), dict(K=0), dict(group=48), dict(group=0),
    dict(y=one), dict(y=ctypes.c_void_p(16 + 4 * 4 * 64 - 4)), dict(bias=ctypes.c_void_p(18)),
    dict(resid=ctypes.c_void_p(17), bf16=1)])
def test_linear_entry_refuses(L, bad):
    assert linear(L, **bad) == -1


def test_pack_entries_refuse(L):
    q = lambda W=one, c=one, s=one, N=4, K=64, g=32: L.pragnosia_fp4_quantize(W, 0, c, s, N, K, g, null)  # noqa: E731
    d = lambda W=one, c=one, s=one, N=4, K=64, g=32: L.pragnosia_fp4_dequantize(c, s, W, 0, N, K, g, null)  # noqa: E731
    for f in (q, d):
        for bad in (dict(W=null), dict(W=odd), dict(c=null), dict(c=odd), dict(s=null), dict(s=odd), dict(N=0),
                    dict(K=4), dict(K=1 << 20), dict(g=16), dict(N=(1 << 26) + 1)):
            assert f(**bad) == -1, bad
    assert linear(L, n=0, x=null, y=null) == 0  # nothing to do


def rule(L, logits=one, history=null, stride=0, n=0, r=1.0, ids=null, values=null, M=0, bstride=0, mask=null, S=0,
         state=null, out=far, tokens=null, ws=null, size=0, B=2, V=100):
    return L.pragnosia_rules(logits, 0, history, stride, n, null, null, null, r, null, 0.0, null, 0.0, ids, values, M,
                             bstride, mask, S, state, out, tokens, ws, size, B, V, null)


@pytest.mark.parametrize("bad", [
    dict(logits=null), dict(logits=odd), dict(out=odd), dict(out=null), dict(tokens=one),
    dict(out=ctypes.c_void_p(32)), dict(r=0.0), dict(n=5),
    dict(n=-1), dict(n=5, history=one, stride=4), dict(n=(1 << 24) + 1, history=one, stride=1 << 30), dict(M=3),
    dict(M=3, ids=one), dict(M=3, ids=one, values=one, bstride=2), dict(M=-1), dict(M=(1 << 20) + 1, ids=one, values=one),
    dict(S=1), dict(S=3, mask=one), dict(S=-1), dict(B=-1), dict(B=1 << 16), dict(V=0), dict(V=(1 << 26) + 1),
    dict(n=1 << 20, history=one, stride=1 << 20, M=1 << 10, ids=one, values=one),
    dict(out=null, tokens=one, V=40000), dict(out=null, tokens=one, V=40000, ws=one, size=79),
    dict(out=null, tokens=one, V=40000, ws=odd, size=1 << 20)])
def test_rules_entry_refuses(L, bad):
    assert rule(L, **bad) == -1


def test_rules_entry_of_no_rows(L):
    assert rule(L, B=0, logits=null) == 0


def test_no_cpu_path():
    with pytest.raises(PragnosiaError, match="no CPU fallback"):
        fp4.quantize(z(16, 64))
    with pytest.raises(PragnosiaError, match="no CPU fallback"):
        fp4.linear(z(2, 64), weight())
    with pytest.raises(PragnosiaError, match="no CPU fallback"):
        fp4.dequantize(weight())
    with pytest.raises(PragnosiaError, match="no CPU fallback"):
        rules.next_token(z(2, 10))
    with pytest.raises(PragnosiaError, match="no CPU fallback"):
        rules.apply_rules(z(2, 10), z(2, 3, **L64))


def weight(N=16, K=64, group=32):
    nbytes, count = fp4._sizes("", N, K, group)
    return fp4.Weight4(z(nbytes, dtype=torch.uint8), z(count, dtype=torch.bfloat16), N, K, group)


@pytest.mark.parametrize("codes,scales,N,K,group,what", [
    (z(1024), z(64), 16, 64, 32, "codes"), (z(1024, dtype=torch.uint8), z(64), 16, 64, 32, "scales"),
    (z(1024, dtype=torch.uint8), z(63, dtype=torch.bfloat16), 16, 64, 32, "scales"),
    (z(2048, dtype=torch.uint8)[::2], z(64, dtype=torch.bfloat16), 16, 64, 32, "codes"),
    (z(1024, dtype=torch.uint8), z(64, dtype=torch.bfloat16), 16, 60, 32, "multiple of 8"),
    (z(1024, dtype=torch.uint8), z(64, dtype=torch.bfloat16), 16, 64, 48, "group")])
def test_weight_refuses(codes, scales, N, K, group, what):
    with pytest.raises(PragnosiaError, match=what):
        fp4.Weight4(codes, scales, N, K, group)


def test_weight_is_immutable():
    Q = weight()
    assert Q.shape == (16, 64) and "Weight4(16, 64" in repr(Q)
    for name in ("codes", "N", "other"):
        with pytest.raises(PragnosiaError, match="cannot be changed"):
            setattr(Q, name, 1)


@pytest.fixture
def unguarded(monkeypatch):
    """The calls below carry a mismatch each, so none gets as far as a launch."""
    for mod in (fp4, rules):
        monkeypatch.setattr(mod, "_require_gpu", lambda *t: None)
        monkeypatch.setattr(mod, "gen_lib", lambda: pytest.fail("a mismatched call reached the C ABI"))


@pytest.mark.parametrize("W,group,what", [
    (z(64), 32, "weight"), (z(2, 64).double(), 32, "fp32 or bf16"), (z(2, 64).half(), 32, "fp32 or bf16"),
    (z(2, 60), 32, "multiple of 8"), (z(0, 64), 32, "N from 1"), (z(2, 0), 32, "N from 1"), (z(2, 64), 16, "group"),
    (z(2, 65544), 32, "65536")])
def test_quantize_refuses(unguarded, W, group, what):
    with pytest.raises(PragnosiaError, match=what):
        fp4.quantize(W, group)


def test_quantize_out_refuses(unguarded):
    for W, group in ((z(17, 64), 32), (z(16, 72), 32), (z(16, 64), 64)):
        with pytest.raises(PragnosiaError, match="out is"):
            fp4.quantize(W, group, out=weight())
    with pytest.raises(PragnosiaError, match="fp32 or bf16"):
        fp4.dequantize(weight(), torch.float16)


LN = torch.nn.LayerNorm


@pytest.mark.parametrize("x,kw,what", [
    (z(2, 72), {}, "x has shape"), (z(2, 64).double(), {}, "fp32 or bf16"), (z(2, 64).long(), {}, "fp32 or bf16"),
    (torch.tensor(1.0), {}, "expected"), (z(2, 64), dict(bias=z(17)), "bias has shape"),
    (z(2, 64), dict(bias=z(16, **L64)), "bias must be"), (z(2, 64), dict(resid=z(3, 16)), "resid"),
    (z(2, 64), dict(resid=z(16)), "resid"), (z(2, 3, 64), dict(resid=z(6, 16)), "resid"),
    (z(2, 64), dict(act="relu"), "gelu"), (z(2, 64), dict(norm=LN(32)), "LayerNorm over 64"),
    (z(2, 64), dict(norm=LN(64, elementwise_affine=False)), "affine"), (z(2, 64), dict(norm=torch.nn.RMSNorm(64)), "affine"),
    (z(2, 64), dict(norm=LN(64, eps=-1.0)), "negative"),
    (torch.empty(1 << 25, 64, device="meta"), {}, "codes is on"), (z(1).expand((1 << 24) + 1, 64), {}, "2\\^24 rows")])
def test_linear_refuses(unguarded, x, kw, what):
    with pytest.raises(PragnosiaError, match=what), torch.no_grad():
        fp4.linear(x, weight(), **kw)


def test_gradients_and_tangents_refused(unguarded):
    import torch.autograd.forward_ad as fwAD
    x = z(2, 64, requires_grad=True)
    for kw in (dict(x=x), dict(x=z(2, 64), bias=z(16, requires_grad=True)), dict(x=z(2, 64), norm=LN(64)),
               dict(x=z(2, 64), resid=z(2, 16, requires_grad=True))):
        with pytest.raises(PragnosiaError, match="no backward"):
            fp4.linear(Q=weight(), **kw)
    with pytest.raises(PragnosiaError, match="no backward"):
        rules.apply_rules(x)
    with pytest.raises(PragnosiaError, match="no backward"):
        rules.next_token(z(2, 10), z(2, 3, **L64), frequency=z(2, requires_grad=True))
    with fwAD.dual_level():
        d = fwAD.make_dual(z(2, 64), z(2, 64))
        for f in (lambda: fp4.linear(d, weight()), lambda: fp4.quantize(d, 32), lambda: rules.next_token(d)):
            with pytest.raises(PragnosiaError, match="forward-mode"):
                f()


H = z(2, 3, **L64)


@pytest.mark.parametrize("kw,what", [
    (dict(logits=z(10)), "logits"), (dict(logits=z(2, 10).half()), "fp32 or bf16"), (dict(logits=z(2, 0)), "words"),
    (dict(logits=z(1).expand(65536, 10)), "65535"), (dict(history=z(3, 3, **L64)), "history has shape"),
    (dict(history=z(2, 3)), "history must be integers"), (dict(lengths=z(2, **L64)), "there is none"),
    (dict(prompt=z(2, **L64)), "there is none"), (dict(history=H, lengths=z(3, **L64)), "lengths has shape"),
    (dict(history=H, lengths=z(2)), "lengths must be integers"), (dict(history=H, prompt=z(2, 1, **L64)), "prompt has shape"),
    (dict(history=z(1, **L64).expand(2, (1 << 24) + 1)), "2\\^24 tokens"),
    (dict(repetition=0.0), "repetition must be"), (dict(repetition=-1.0), "repetition must be"),
    (dict(repetition=float("inf")), "finite"), (dict(presence=float("nan")), "presence must be finite"),
    (dict(frequency=z(3)), "frequency has shape"), (dict(presence=z(2, **L64)), "presence must be floating"),
    (dict(bias=(z(3, 4, **L64), z(3, 4))), "bias ids"), (dict(bias=(z(4), z(4))), "bias ids must be integers"),
    (dict(bias=(z(2, 4, **L64), z(4))), "bias_values has shape"), (dict(bias=(z(4, **L64), z(4, **L64))), "floating"),
    (dict(bias=(z(1, **L64).expand((1 << 20) + 1), z(1).expand((1 << 20) + 1))), "2\\^20"),
    (dict(history=z(1, **L64).expand(2, 1 << 20), bias=(z(1 << 10, **L64), z(1 << 10))), "31 bits"),
    (dict(bias=(z(4, **L64), None)), "ids, values"), (dict(state=z(2, **L64)), "there is none"),
    (dict(mask=z(2, 2, dtype=torch.int32)), "mask has shape"), (dict(mask=z(2, 1)), "mask"),
    (dict(mask=z(0, 1, dtype=torch.int32)), "S > 0"), (dict(mask=z(3, 1, dtype=torch.int32)), "without a state"),
    (dict(mask=z(3, 1, dtype=torch.int32), state=z(2)), "state must be integers"),
    (dict(mask=z(3, 1, dtype=torch.int32), state=z(3, **L64)), "state has shape")])
def test_rules_refuse(unguarded, kw, what):
    kw = dict(logits=z(2, 10)) | kw
    for f in (rules.next_token, rules.apply_rules):
        with pytest.raises(PragnosiaError, match=what):
            f(**kw)


def tail(L, tokens=one, history=null, stride=0, cap=0, lengths=null, next=null, S=0, state=null, emb=null, d=0, ctx=0,
         ctr=(one, far), pos=(one, far), tok=far, h=far, B=2, V=100):
    return L.pragnosia_rules_tail(tokens, history, stride, cap, lengths, next, S, state, emb, emb, d, ctx, *ctr, *pos, far,
                                  9, tok, h, null, 0, B, V, null)


@pytest.mark.parametrize("bad", [
    dict(), dict(tokens=null, history=one, stride=4, cap=4, lengths=one), dict(history=one, stride=4, cap=4),
    dict(lengths=one), dict(history=one, stride=3, cap=4, lengths=one), dict(history=one, lengths=one), dict(next=one, S=3),
    dict(state=one), dict(next=one, state=one), dict(emb=one, ctx=4), dict(emb=one, d=8), dict(emb=one, d=8, ctx=4, h=null),
    dict(emb=one, d=8, ctx=4, ctr=(one, one)), dict(emb=one, d=8, ctx=4, pos=(far, far)), dict(emb=one, d=8, ctx=4, tok=one),
    dict(next=one, state=one, S=3, B=-1), dict(next=one, state=one, S=3, V=0)])
def test_tail_entry_refuses(L, bad):
    assert tail(L, **bad) == -1


def test_tail_entry_of_no_rows(L):
    assert tail(L, tokens=null, next=one, state=one, S=3, B=0) == 0


@pytest.mark.parametrize("kw,what", [
    (dict(vocab=10), "either pair"), (dict(history=H, lengths=z(2, **L64)), "vocabulary's size"),
    (dict(history=H, vocab=10), "either pair"), (dict(history=H, lengths=z(3, **L64), vocab=10), "lengths has shape"),
    (dict(history=H, lengths=z(2, dtype=torch.int32), vocab=10), "lengths must be int64"),
    (dict(history=z(3, 2, **L64).t(), lengths=z(2, **L64), vocab=10), "history must be int64 and dense"),
    (dict(history=H[:, :0], lengths=z(2, **L64), vocab=10), "no room"), (dict(next=z(3, 10, dtype=torch.int32)), "either pair"),
    (dict(next=z(3, 10, **L64), state=z(2, **L64)), "dense int32"), (dict(next=z(0, 10, dtype=torch.int32), state=z(2, **L64)),
                                                                     "S > 0"),
    (dict(next=z(3, 10, dtype=torch.int32), state=z(2)), "state must be int64")])
def test_advance_refuses(unguarded, kw, what):
    with pytest.raises(PragnosiaError, match=what):
        rules.advance(z(2, **L64), **kw)


def test_weights_are_copied_and_saved(tmp_path):
    codes = torch.arange(2048, dtype=torch.int64).to(torch.uint8)
    Q = fp4.Weight4(codes, torch.arange(64).bfloat16(), 20, 128, 64, torch.bfloat16)
    m = torch.nn.Module()
    m.q = Q
    for R in (copy.copy(Q), copy.deepcopy(m).q, pickle.loads(pickle.dumps(Q))):
        assert R is not Q and (R.N, R.K, R.group, R.dtype) == (20, 128, 64, torch.bfloat16)
        assert torch.equal(R.codes, Q.codes) and torch.equal(R.scales, Q.scales)
    torch.save(Q, tmp_path / "q.pt")
    with torch.serialization.safe_globals([fp4.Weight4]):
        R = torch.load(tmp_path / "q.pt", weights_only=True)
    assert torch.equal(R.codes, Q.codes) and R.shape == Q.shape
