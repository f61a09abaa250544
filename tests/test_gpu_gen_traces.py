"""Generation's operators on GPU tensors, compiled whole, traced and exported: the graph holds the custom op, and what it
computes is the eager call's."""
import pytest
import torch
from torch.fx.experimental.proxy_tensor import make_fx

from pragnosia_amd import fp4, rules

pytestmark = pytest.mark.gpu
DEV = "cuda"
N, K, n, B, V, L = 48, 136, 5, 3, 501, 40


def operands(seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device=DEV)  # noqa: E731
    i = lambda hi, *s: torch.randint(0, hi, s, generator=g, device=DEV)  # noqa: E731
    mask = i(1 << 32, 4, (V + 31) // 32).to(torch.int32)
    return (r(N, K), r(n, K), r(N), r(n, N), 3 * r(B, V), i(V, B, L), i(L + 1, B), 1 + r(B).abs(), mask, i(5, B) - 1)


W0 = torch.randn(N, K, generator=torch.Generator().manual_seed(7))
KEPT = {}


def kept():
    """A weight and a norm made before the trace, as a model has them."""
    if not KEPT:
        ln = torch.nn.LayerNorm(K, device=DEV).requires_grad_(False)
        ln.weight.copy_(1 + 0.1 * torch.randn(K, generator=torch.Generator().manual_seed(8)))
        KEPT.update(Q=fp4.quantize(W0.to(DEV), 32), ln=ln)
    return KEPT


def quantize(W, *rest):
    Q = fp4.quantize(W, 32)
    return Q.codes, Q.scales


def round_trip(W, *rest):
    return fp4.dequantize(fp4.quantize(W, 64))


def dequantize(W, *rest):
    return fp4.dequantize(kept()["Q"]) + W


def linear(W, x, bias, resid, *rest):
    return fp4.linear(x, kept()["Q"], bias, norm=kept()["ln"], act="gelu", resid=resid)


def next_token(W, x, bias, resid, logits, history, lengths, repetition, mask, state):
    return rules.next_token(logits, history, lengths, repetition=repetition, presence=0.5, mask=mask, state=state)


def apply_rules(W, x, bias, resid, logits, history, lengths, repetition, mask, state):
    return rules.apply_rules(logits, history, lengths, repetition=1.5, frequency=repetition, mask=mask, state=state)


CALLS = [(quantize, "fp4_quantize"), (round_trip, "fp4_dequantize"), (dequantize, "fp4_dequantize"), (linear, "fp4_linear"),
         (next_token, "rules_token"), (apply_rules, "rules_apply")]
each = pytest.mark.parametrize("f,op", CALLS, ids=[f.__name__ for f, _ in CALLS])


def same(a, b):
    a, b = (list(t) if isinstance(t, tuple) else [t] for t in (a, b))
    assert len(a) == len(b) and all(torch.equal(u, v) and u.dtype == v.dtype for u, v in zip(a, b))


@each
@pytest.mark.parametrize("dynamic", [False, True])
def test_compiled_whole(f, op, dynamic):
    kept()
    torch._dynamo.reset()
    names = []

    def backend(gm, inputs):
        names.append(gm.print_readable(print_output=False))
        return gm.forward

    call = torch.compile(f, backend=backend, fullgraph=True, dynamic=dynamic)
    for seed in (0, 1):
        same(call(*operands(seed)), f(*operands(seed)))
    assert len(names) == 1 and f"pragnosia_gen.{op}" in names[0]
    same(torch.compile(f, backend="aot_eager", fullgraph=True, dynamic=dynamic)(*operands()), f(*operands()))


@each
@pytest.mark.parametrize("mode", ["real", "fake", "symbolic"])
def test_make_fx(f, op, mode):
    kept()
    traced = make_fx(f, tracing_mode=mode, _allow_non_fake_inputs=True)(*operands())
    assert op in traced.code
    for seed in (0, 1):
        same(traced(*operands(seed)), f(*operands(seed)))


@each
@pytest.mark.filterwarnings("ignore::torch.jit.TracerWarning")
def test_jit_trace(f, op):
    kept()
    traced = torch.jit.trace(f, operands(), check_trace=False)
    assert f"pragnosia_gen::{op}" in str(traced.graph)
    for seed in (0, 1):
        same(traced(*operands(seed)), f(*operands(seed)))
