"""CPU checks of the language model's ends under torch's traces and modes: what records or replaces torch's operations
sees the custom ops, and a forward-mode tangent is refused. Nothing is launched: the calls into the library are left
out, so results hold anything and only their shapes and the record are looked at."""
import contextlib

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.autograd import forward_ad
from torch.fx.experimental.proxy_tensor import make_fx
from torch.utils._python_dispatch import TorchDispatchMode

from pragnosia_amd import embed, head
from pragnosia_amd._lib import PragnosiaError

n, V, d, K = 6, 11, 16, 3


@pytest.fixture(autouse=True)
def calls(monkeypatch):
    """The library's calls that were made, by name."""
    made = []
    for mod in (head, embed):
        monkeypatch.setattr(mod, "_require_gpu", lambda *t: None)
        monkeypatch.setattr(mod, "_call", lambda what, fn, t, *args: made.append((what, args)))
    return made


def operands(grad=False):
    h, W = torch.randn(n, d).bfloat16().requires_grad_(grad), torch.randn(V, d).requires_grad_(grad)
    return h, W, torch.randint(0, V, (n,)), torch.randint(0, V, (n, K)), torch.randn(n, K)


def ce(h, W, y, ids, z):
    return head.linear_cross_entropy(h, W, y)


def kd(h, W, y, ids, z):
    return head.linear_distill(h, W, ids, z, 2.0, y)


def kd_alone(h, W, y, ids, z):
    return head.linear_distill(h, W, ids, z, 2.0)[0]


def rows(h, W, y, ids, z):
    return embed.embedding(ids, W, 0.5)


CALLS = [(ce, "head_loss"), (kd, "head_loss"), (kd_alone, "head_loss"), (rows, "embed")]


def recorded(graph):
    return [str(node.target) for node in graph.graph.nodes if node.op == "call_function"]


def _flat(out):
    return [t for t in (out if isinstance(out, tuple) else (out,)) if t is not None]


@pytest.mark.parametrize("f,op", CALLS)
@pytest.mark.parametrize("mode", ["real", "fake", "symbolic", "pre_dispatch"])
def test_make_fx_records_the_op(f, op, mode):
    kw = dict(pre_dispatch=True) if mode == "pre_dispatch" else dict(tracing_mode=mode)
    got = recorded(make_fx(f, **kw)(*operands()))
    assert any(t.startswith(f"pragnosia_lm.{op}.") for t in got) and not any("empty" in t for t in got), got


@pytest.mark.parametrize("f,op", CALLS)
def test_make_fx_records_the_gradient(f, op):
    def both(h, W, y, ids, z):
        out = f(h, W, y, ids, z)
        loss = sum(t.sum() for t in (out if isinstance(out, tuple) else (out,)))
        return torch.autograd.grad(loss, [W] if f is rows else [h, W])

    got = recorded(make_fx(both)(*operands(True)))
    assert any(t.startswith(f"pragnosia_lm.{op}_bwd.") for t in got) and not any("empty.mem" in t for t in got), got


@pytest.mark.parametrize("f,op", CALLS)
def test_make_fx_of_the_backward_alone(f, op, calls):
    """A graph built by an eager call, its backward traced."""
    h, W, *rest = operands(True)
    out = f(h, W, *rest)
    out = out[0] if isinstance(out, tuple) else out
    assert [c[0] for c in calls] == [f"pragnosia_{'embed' if f is rows else 'head'}_fwd"]
    traced = make_fx(lambda g: torch.autograd.grad(out, [W] if f is rows else [h, W], g))(torch.randn_like(out))
    got = recorded(traced)
    assert any(t.startswith(f"pragnosia_lm.{op}_bwd.") for t in got) and not any("empty.mem" in t for t in got), got


@pytest.mark.parametrize("f,op", CALLS)
def test_jit_trace_records_the_op(f, op):
    traced = torch.jit.trace(f, operands(), check_trace=False)
    assert f"pragnosia_lm::{op}" in str(traced.graph) and "aten::empty" not in str(traced.graph)


@pytest.mark.parametrize("f,op", CALLS)
def test_fake_tensors(f, op, calls):
    """Shapes and types from the ops' fakes, inside the mode and with its tensors outside it."""
    want = [tuple(t.shape) for t in _flat(f(*operands()))]
    calls.clear()
    with FakeTensorMode() as mode:
        fakes = operands(True)
        inside = _flat(f(*fakes))
    outside = _flat(f(*fakes))
    for got in (inside, outside):
        assert [tuple(t.shape) for t in got] == want and all(t.fake_mode is mode for t in got)
    outside[0].float().sum().backward()
    assert fakes[1].grad.shape == (V, d) and fakes[1].grad.dtype == torch.float32
    assert not calls  # nothing of theirs reached the library


class Watch(TorchDispatchMode):
    def __init__(self):
        super().__init__()
        self.seen = []

    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        self.seen.append(str(func))
        return func(*args, **(kwargs or {}))


@pytest.mark.parametrize("f,op", CALLS)
@pytest.mark.parametrize("grad", [False, True])
def test_dispatch_mode_sees_the_op(f, op, grad):
    args = operands(grad)
    with Watch() as watch:
        out = _flat(f(*args))[0]
        if grad:
            out.float().sum().backward()
    assert f"pragnosia_lm.{op}.default" in watch.seen and not any("aten.empty" in s for s in watch.seen)
    assert (f"pragnosia_lm.{op}_bwd.default" in watch.seen) == grad


@pytest.mark.parametrize("f,op", CALLS)
@pytest.mark.parametrize("grad", [False, True])
def test_gradient_types_of_a_watched_backward(f, op, grad):
    """The traced backward of an eager graph gives the eager one's shapes and types, fp32 and bf16 operands alike."""
    for th, tw in ((torch.float32, torch.float32), (torch.float32, torch.bfloat16), (torch.bfloat16, torch.float32)):
        h, W, *rest = operands()
        h, W = h.to(th).requires_grad_(grad), W.to(tw).requires_grad_()
        out = _flat(f(h, W, *rest))[0]
        leaves = [W] if f is rows or not grad else [h, W]
        g = torch.randn(out.shape, dtype=out.dtype)
        want = torch.autograd.grad(out, leaves, g, retain_graph=True)
        with Watch():
            got = torch.autograd.grad(out, leaves, g)
        for a, b, leaf in zip(got, want, leaves):
            assert a.dtype == b.dtype == leaf.dtype and a.shape == b.shape == leaf.shape


def test_an_eager_call_is_direct(calls):
    """Without a mode or a trace the library is called from an autograd function, parameters and modules included."""
    h, W, *rest = operands()
    for t in (W, torch.nn.Parameter(W)):
        for f, _ in CALLS:
            calls.clear()
            out = _flat(f(h, t, *rest))[0]
            assert len(calls) == 1
            names = set()
            node = out.grad_fn
            while node is not None:
                names.add(node.name())
                node = node.next_functions[0][0] if node.next_functions else None
            if t is not W:
                assert names & {"_HeadLossBackward", "_EmbeddingBackward"}, names


OPS = [lambda h, W, y, ids, z: torch.ops.pragnosia_lm.head_loss(h, W, y, ids, z, 2.0),
       lambda h, W, y, ids, z: torch.ops.pragnosia_lm.embed(y, W, 1.0, False)]


@pytest.mark.parametrize("f", [f for f, _ in CALLS] + OPS)
def test_tangents_are_refused(f):
    """A dual tensor raises, whether it requires a gradient or not, and whichever operand it is; without a tangent a
    forward-mode level changes nothing. (The table of ids and the teacher's logits have none to lose.)"""
    h, W, *rest = operands()
    with forward_ad.dual_level():
        plain = _flat(f(h, W, *rest))
        assert all(forward_ad.unpack_dual(t).tangent is None for t in plain if t.is_floating_point())
        for which in (0, 1):
            if which == 0 and (f is rows or f is OPS[1]):
                continue
            for grad in (False, True):
                pair = [h.clone().requires_grad_(grad), W.clone().requires_grad_(grad)]
                pair[which] = forward_ad.make_dual(pair[which], torch.ones_like(pair[which]))
                with pytest.raises((PragnosiaError, NotImplementedError), match="forward"):
                    f(*pair, *rest)


@pytest.mark.parametrize("f,op", CALLS)
def test_tangents_of_a_gradient_are_refused(f, op):
    h, W, *rest = operands(True)
    out = _flat(f(h, W, *rest))[0]
    with forward_ad.dual_level():
        g = forward_ad.make_dual(torch.ones_like(out), torch.ones_like(out))
        with pytest.raises(PragnosiaError, match="forward"):
            torch.autograd.grad(out, W, g)


@pytest.mark.parametrize("f,op", CALLS)
def test_transforms_are_refused(f, op):
    """torch.func's transforms raise."""
    h, W, *rest = operands()
    call = lambda w: _flat(f(h, w, *rest))[0].sum()
    for run in (lambda: torch.func.jvp(call, (W,), (W,)), lambda: torch.func.grad(call)(W),
                lambda: torch.func.vmap(call)(W.expand(2, V, d))):
        with pytest.raises((RuntimeError, NotImplementedError)):
            run()


@pytest.mark.parametrize("f,op", CALLS)
@pytest.mark.parametrize("way", ["eager", "mode", "compiled"])
def test_empty_batch(f, op, way):
    """No tokens: empty results, and gradients of zeros, by every way."""
    h, W, *rest = operands()
    h, W = h[:0].clone().requires_grad_(), W.requires_grad_()
    rest = [t[:0] for t in rest]
    if way == "compiled":
        torch._dynamo.reset()
        f = torch.compile(f, backend="aot_eager", fullgraph=True)
    watch = Watch()
    with watch if way == "mode" else contextlib.nullcontext():
        out = _flat(f(h, W, *rest))
        assert all(t.shape[0] == 0 for t in out)
        sum(t.float().sum() for t in out).backward()
    if op == "head_loss":
        assert h.grad.shape == (0, d) and W.grad.shape == (V, d) and not W.grad.any()
    assert W.grad.dtype == W.dtype and W.grad.shape == W.shape
