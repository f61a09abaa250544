"""CPU checks of generation's operators under torch's traces and modes: what records or replaces torch's operations sees the
custom ops. Nothing is launched: the calls into the library are left out, so results hold anything and only their shapes
and the record are looked at."""
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.fx.experimental.proxy_tensor import make_fx
from torch.utils._python_dispatch import TorchDispatchMode

from pragnosia_amd import fp4, rules

N, K, n, G, B, V, L, M, S = 40, 136, 5, 32, 3, 70, 9, 4, 6


@pytest.fixture(autouse=True)
def calls(monkeypatch):
    """The library's calls that were made, by name."""
    made = []
    for mod in (fp4, rules):
        monkeypatch.setattr(mod, "_require_gpu", lambda *t: None)
        monkeypatch.setattr(mod, "_call", lambda what, fn, t, *args: made.append(what))
    return made


def operands(**where):
    """Of every call below, on the CPU or where said."""
    z, i = (lambda *s: torch.zeros(*s, **where)), (lambda *s: torch.zeros(*s, dtype=torch.long, **where))
    nbytes, count = fp4._sizes("", N, K, G)
    return (z(N, K), z(n, K), torch.zeros(nbytes, dtype=torch.uint8, **where),
            torch.zeros(count, dtype=torch.bfloat16, **where), z(K), z(K), z(N), z(n, N), z(B, V), i(B, L), i(B), z(B),
            i(M), z(M), torch.zeros(S, (V + 31) // 32, dtype=torch.int32, **where), i(B))


def weight4(codes, scales):
    return fp4.Weight4.__new__(fp4.Weight4)._set(codes, scales, N, K, G, torch.float32)


def layer_norm(w, b):
    with FakeTensorMode(allow_non_fake_inputs=True):
        m = torch.nn.LayerNorm(K)
    m.weight, m.bias = (torch.nn.Parameter(t, requires_grad=False) for t in (w, b))
    return m


def quantize(W, *rest):
    Q = fp4.quantize(W, G)
    return Q.codes, Q.scales


def dequantize(W, x, codes, scales, *rest):
    return fp4.dequantize(weight4(codes, scales))


def round_trip(W, *rest):
    return fp4.dequantize(fp4.quantize(W, G))


def linear(W, x, codes, scales, w, b, bias, resid, *rest):
    return fp4.linear(x, weight4(codes, scales), bias, act="gelu", resid=resid)


def by_rules(call, listed=False):
    def f(W, x, codes, scales, w, b, bias, resid, logits, history, lengths, repetition, ids, values, mask, state):
        return call(logits, history, lengths, repetition=repetition, presence=0.5, bias=(ids, values) if listed else None,
                    mask=mask, state=state)
    return f


CALLS = [(quantize, "fp4_quantize"), (dequantize, "fp4_dequantize"), (round_trip, "fp4_dequantize"), (linear, "fp4_linear"),
         (by_rules(rules.next_token), "rules_token"), (by_rules(rules.apply_rules), "rules_apply"),
         (by_rules(rules.next_token, True), "rules_token"), (by_rules(rules.apply_rules, True), "rules_apply")]
each = pytest.mark.parametrize("f,op", CALLS, ids=["quantize", "dequantize", "round_trip", "linear", "next_token", "apply_rules",
                                                   "next_token_listed", "apply_rules_listed"])


def flat(out):
    return list(out) if isinstance(out, tuple) else [out]


@each
@pytest.mark.parametrize("mode", ["real", "fake", "symbolic", "pre_dispatch"])
def test_make_fx_records_the_op(f, op, mode):
    kw = dict(pre_dispatch=True) if mode == "pre_dispatch" else dict(tracing_mode=mode)
    graph = make_fx(f, **kw)(*operands()).graph
    got = [str(node.target) for node in graph.nodes if node.op == "call_function"]
    assert any(t.startswith(f"pragnosia_gen.{op}.") for t in got) and not any("empty" in t for t in got), got


@each
@pytest.mark.parametrize("device", ["cpu", "cuda"])
def test_fake_tensors(f, op, device, calls):
    """Shapes and types from the ops' fakes, inside the mode and with its tensors outside it; no device is asked for."""
    want = [(tuple(t.shape), t.dtype) for t in flat(f(*operands()))]
    calls.clear()
    with FakeTensorMode() as mode:
        fakes = operands(device=device)
        inside = flat(f(*fakes))
    outside = flat(f(*fakes))
    for got in (inside, outside):
        assert [(tuple(t.shape), t.dtype) for t in got] == want
        assert all(t.fake_mode is mode and t.device.type == device for t in got)
    assert not calls


def test_fake_norm():
    """A norm's parameters as fake tensors."""
    with FakeTensorMode():
        W, x, codes, scales, w, b, *rest = operands(device="cuda")
        y = fp4.linear(x, weight4(codes, scales), norm=layer_norm(w, b))
    assert y.shape == (n, N) and y.device.type == "cuda"


class Watch(TorchDispatchMode):
    def __init__(self):
        super().__init__()
        self.seen = []

    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        self.seen.append(str(func))
        return func(*args, **(kwargs or {}))


@each
def test_modes_see_the_op(f, op):
    with Watch() as w:
        f(*operands())
    assert any(s.startswith(f"pragnosia_gen.{op}.") for s in w.seen), w.seen


@each
@pytest.mark.filterwarnings("ignore::torch.jit.TracerWarning")
def test_jit_trace_records_the_op(f, op):
    traced = torch.jit.trace(f, operands(), check_trace=False)
    assert f"pragnosia_gen::{op}" in str(traced.graph) and "aten::empty" not in str(traced.graph)


@each
@pytest.mark.parametrize("dynamic", [False, True])
def test_compiles_whole(f, op, dynamic):
    torch._dynamo.reset()
    graphs = []

    def backend(gm, inputs):
        graphs.append(gm)
        return gm.forward

    got = torch.compile(f, backend=backend, fullgraph=True, dynamic=dynamic)(*operands())
    assert [tuple(t.shape) for t in flat(got)] == [tuple(t.shape) for t in flat(f(*operands()))]
    assert len(graphs) == 1 and f"pragnosia_gen.{op}" in graphs[0].print_readable(print_output=False)


def test_a_weight_leaves_a_compiled_function():
    """Whole, and as immutable as one of an eager call."""
    torch._dynamo.reset()
    W = operands()[0]
    Q = torch.compile(lambda W: fp4.quantize(W, G), backend="eager", fullgraph=True)(W)
    assert type(Q) is fp4.Weight4 and (Q.N, Q.K, Q.group, Q.dtype) == (N, K, G, torch.float32)
    assert Q.codes.shape == (fp4._sizes("", N, K, G)[0],)
    with pytest.raises(fp4.PragnosiaError, match="cannot be changed"):
        Q.N = 3
    y = torch.compile(lambda x, Q: fp4.linear(x, Q), backend="eager", fullgraph=True)(operands()[1], Q)
    assert y.shape == (n, N)


def test_exported():
    class Layer(torch.nn.Module):
        def forward(self, x, codes, scales):
            return fp4.linear(x, weight4(codes, scales))

    W, x, codes, scales, *rest = operands()
    got = torch.export.export(Layer(), (x, codes, scales)).graph_module.code
    assert "fp4_linear" in got


def test_marks_of_31_bits():
    """The comparisons are those of the lengths in bits."""
    sizes = sorted({v for k in range(25) for v in ((1 << k) - 1, 1 << k, (1 << k) + 1) if v <= 1 << 24})
    for L in sizes:
        for M in sizes:
            if M <= 1 << 20:
                assert rules._marks_fit(L, M) == (L.bit_length() + M.bit_length() <= 31), (L, M)
