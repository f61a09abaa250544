"""Rules for the next token, on hand-written kernels (csrc/rules.hip; C ABI in pragnosia_amd/include/pragnosia_gen.h): penalties
for repeated tokens, biases of some words, masks of what a grammar allows, in one pass over the logits.

    token = next_token(logits, history, lengths, prompt, repetition=1.2, bias=(ids, values), mask=mask, state=state)
    logits = apply_rules(logits, ...)           # the same rules, the logits for a sampler of the caller's own
    advance(token, history, lengths, next, state)    # the token joins the history and moves the grammar's state, in place

For row b and word v, in fp32, each step rounded:

    a word among history[b, :lengths[b]]                x = l / repetition where l > 0, else l * repetition
    c > 0 times among history[b, prompt[b]:lengths[b]]  x = x - presence, then x = x - frequency * c
    a word of the row's bias list                       x = x + its value
    a word whose mask bit is clear                      x = -inf

`GreedyDecoder(..., rules=TokenRules(...))` chooses its tokens under them; the reference takes the argmax or samples the
logits as they are (`src/bench.py:83`).
"""
from __future__ import annotations

import dataclasses
from typing import Optional, Union

import torch
from torch import Tensor

from ._lib import PragnosiaError, check, gen_lib
from .fp4 import _device, _fits, _quiet
from .head import _BF16, _F32, _FLOATS, _I64, _INTS, _as, _at, _call, _no_tangents, _raw_stream, _watched
from .ops import _expect, _require_gpu

Penalty = Union[float, Tensor]
_MAX, _TINY = torch.finfo(torch.float32).max, 2.0 ** -149  # of what the kernels take a penalty's number in


def _in_range(name: str, p: float) -> bool:
    """Whether fp32 holds a penalty: finite, and above 0 where it divides. (1e39 is finite here and infinite there, and its
    product with a logit of 0 a NaN, which is above every word.)"""
    return _TINY <= p <= _MAX if name == "repetition" else -_MAX <= p <= _MAX


def _marks_fit(L: int, M: int) -> bool:
    """Whether a history of L (up to 2^24) and a list of M (up to 2^20) entries have 31 bits together at most, by comparisons
    alone: in a trace a size is no Python number and has no bit_length."""
    return not any(M >= 1 << k - 1 and L >= 1 << 31 - k for k in range(7, 22))


def _out_of_range(what: str, name: str, p: float) -> PragnosiaError:
    return PragnosiaError(f"{what}: {name} must be finite{' and above 0' if name == 'repetition' else ''} in fp32, got {p}")


def _checked(op: str, logits: Tensor, history: Optional[Tensor], lengths: Optional[Tensor], prompt: Optional[Tensor],
             penalties, ids: Optional[Tensor], values: Optional[Tensor], mask: Optional[Tensor],
             state: Optional[Tensor]) -> None:
    """Refuses what the kernels do not take; penalties: three of (name, number or (B,) tensor)."""
    _require_gpu(logits, history, lengths, prompt, ids, values, mask, state,
                 *(p for _, p in penalties if isinstance(p, Tensor)))
    if logits.dim() != 2 or logits.dtype not in _FLOATS:
        raise PragnosiaError(f"{op}: logits (B, V) in fp32 or bf16 expected, got {tuple(logits.shape)} {logits.dtype}")
    (B, V), dev = logits.shape, logits.device
    if not 0 < V <= 1 << 26 or B > 65535:
        raise PragnosiaError(f"{op}: at most 65535 rows of 1 to 2^26 words, got {B} of {V}")
    _expect(op, dev, history=(history, (B, None)), lengths=(lengths, (B,)), prompt=(prompt, (B,)), state=(state, (B,)))
    for name, t in (("history", history), ("lengths", lengths), ("prompt", prompt), ("state", state), ("bias ids", ids)):
        if t is not None and t.dtype not in _INTS:
            raise PragnosiaError(f"{op}: {name} must be integers, got {t.dtype}")
    if history is None and (lengths is not None or prompt is not None):
        raise PragnosiaError(f"{op}: lengths and prompt say how a history is read; there is none")
    if history is not None and history.shape[1] > 1 << 24:
        raise PragnosiaError(f"{op}: at most 2^24 tokens of history, got {history.shape[1]}")
    for name, p in penalties:
        if isinstance(p, Tensor):
            _expect(op, dev, **{name: (p, (B,))})
            if not p.is_floating_point():
                raise PragnosiaError(f"{op}: {name} must be floating, got {p.dtype}")
        elif not _in_range(name, p):
            raise _out_of_range(op, name, p)
    if (ids is None) != (values is None):
        raise PragnosiaError(f"{op}: bias is (ids, values)")
    if ids is not None:
        if ids.dim() not in (1, 2) or (ids.dim() == 2 and ids.shape[0] != B) or ids.shape[-1] > 1 << 20:
            raise PragnosiaError(f"{op}: bias ids (M) or ({B}, M) with M up to 2^20 expected, got {tuple(ids.shape)}")
        _expect(op, dev, bias_ids=(ids, tuple(ids.shape)), bias_values=(values, tuple(ids.shape)))
        if history is not None and not _marks_fit(history.shape[1], ids.shape[-1]):
            raise PragnosiaError(f"{op}: the lengths of history and bias list must have 31 bits together at most, got "
                                 f"{history.shape[1]} and {ids.shape[-1]}")
        if not values.is_floating_point():
            raise PragnosiaError(f"{op}: bias values must be floating, got {values.dtype}")
    words = (V + 31) // 32
    if mask is None:
        if state is not None:
            raise PragnosiaError(f"{op}: state names a line of the mask; there is none")
    else:
        _expect(op, dev, mask=(mask, (None, words)))
        if mask.dtype != torch.int32 or mask.shape[0] == 0:
            raise PragnosiaError(f"{op}: mask (S, {words}) int32 with S > 0 expected, got {tuple(mask.shape)} {mask.dtype}")
        if state is None and mask.shape[0] not in (1, B):
            raise PragnosiaError(f"{op}: without a state the mask has one line or one for each of {B} rows, got "
                                 f"{mask.shape[0]}")


def _launch(logits: Tensor, history: Optional[Tensor], lengths: Optional[Tensor], prompt: Optional[Tensor], penalties,
            ids: Optional[Tensor], values: Optional[Tensor], mask: Optional[Tensor], state: Optional[Tensor],
            out: Optional[Tensor], tokens: Optional[Tensor]) -> None:
    """The C call; penalties: three numbers or (B,) tensors."""
    B, V = logits.shape
    if B == 0:
        return
    L = stride = M = bias_stride = S = 0
    if history is not None and history.shape[1]:
        if history.dtype is not _I64 or history.stride(1) != 1 or (B > 1 and history.stride(0) < history.shape[1]):
            history = history.to(_I64).contiguous()
        L, stride = history.shape[1], max(history.stride(0), history.shape[1])
    args = []
    for p, neutral in zip(penalties, (1.0, 0.0, 0.0)):
        t = _as(p, _F32) if isinstance(p, Tensor) else None
        args += [t, neutral if t is not None else float(p)]
    if ids is not None and ids.shape[-1]:
        ids, values = _as(ids, _I64), _as(values, _F32)
        M = ids.shape[-1]
        bias_stride = M if ids.dim() == 2 else 0
    if mask is not None:
        mask, state, S = _as(mask, torch.int32), _as(state, _I64), mask.shape[0]
    lengths, prompt = _as(lengths, _I64), _as(prompt, _I64)
    nbytes = _gen_workspace(B, V) if tokens is not None else 0
    ws = torch.empty(nbytes, device=logits.device, dtype=torch.uint8) if nbytes else None
    _call("pragnosia_rules", gen_lib().pragnosia_rules, logits, _at(logits), logits.dtype is _BF16, _at(history) if L else
          None, stride, L, _at(lengths), _at(prompt), _at(args[0]), args[1], _at(args[2]), args[3], _at(args[4]), args[5],
          _at(ids) if M else None, _at(values) if M else None, M, bias_stride, _at(mask), S, _at(state), _at(out),
          _at(tokens), _at(ws), nbytes, B, V)


_sizes: dict = {}


def _gen_workspace(B: int, V: int) -> int:
    got = _sizes.get((B, V))
    if got is None:
        got = gen_lib().pragnosia_rules_workspace_bytes(B, V)
        if got < 0:
            raise PragnosiaError(f"pragnosia_rules_workspace_bytes: sizes {(B, V)} rejected")
        if len(_sizes) > 4096:
            _sizes.clear()
        _sizes[B, V] = got
    return got


def _rules(op: str, logits, history, lengths, prompt, repetition, presence, frequency, bias, mask, state, choose: bool):
    ids, values = (None, None) if bias is None else bias
    penalties = (("repetition", repetition), ("presence", presence), ("frequency", frequency))
    floats = [logits, values] + [p for _, p in penalties if isinstance(p, Tensor)]
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in floats):
        raise PragnosiaError(f"{op}: rules have no backward; call it under torch.no_grad()")
    _no_tangents(op, *floats)
    got = _plain(logits, history, lengths, prompt, (repetition, presence, frequency), ids, values, mask, state, choose)
    if got is not None:
        return got
    _checked(op, logits, history, lengths, prompt, penalties, ids, values, mask, state)
    if _watched(*floats, history, lengths, prompt, ids, mask, state):
        # (the ops take penalties as tensors or numbers, and bias as two tensors)
        t = [p if isinstance(p, Tensor) else None for _, p in penalties]
        v = [1.0 if isinstance(p, Tensor) else float(p) for _, p in penalties]
        call = rules_token if choose else rules_apply
        return call(logits, history, lengths, prompt, t[0], v[0], t[1], v[1], t[2], v[2], ids, values, mask, state)
    return _run(logits, history, lengths, prompt, (repetition, presence, frequency), ids, values, mask, state, choose)


def _plain(logits, history, lengths, prompt, penalties, ids, values, mask, state, choose: bool) -> Optional[Tensor]:
    """The usual call, all of whose tensors the kernels take as they are: no conversions, and no refusals to look for, which
    is most of what the host does in the general path (19 us for one row with a history; this one 11). None: not such a
    call."""
    if logits.dim() != 2 or not _quiet({type(t) for t in (logits, history, lengths, prompt, *penalties, ids, values, mask,
                                                          state)}):
        return None
    (B, V), index, dt = logits.shape, logits.get_device(), logits.dtype
    if not (logits.is_cuda and 0 < B <= 65535 and 0 < V <= 1 << 26 and dt in _FLOATS and index == _device()
            and logits.is_contiguous() and not logits.data_ptr() & 15):
        return None
    row = (B,)
    L = stride = M = bias_stride = S = 0
    if history is not None:
        if not (history.dim() == 2 and history.dtype is _I64 and history.get_device() == index and history.shape[0] == B):
            return None
        L, (stride, inner) = history.shape[1], history.stride()
        if inner != 1 or not 0 < L <= 1 << 24 or stride < L:
            return None
        for t in (lengths, prompt):
            if t is not None and not _fits(t, _I64, index, row):
                return None
    elif lengths is not None or prompt is not None:
        return None
    args = []
    for p in penalties:
        if isinstance(p, Tensor):
            if not _fits(p, _F32, index, row):
                return None
            args += [p.data_ptr(), 1.0]
        else:
            args += [None, p]
    if not (isinstance(args[1], float) and _TINY <= args[1] <= _MAX and -_MAX <= args[3] <= _MAX
            and -_MAX <= args[5] <= _MAX):
        return None
    if ids is not None:
        M = ids.shape[-1] if ids.dim() else 0
        shape = row + (M,) if ids.dim() == 2 else (M,)
        if not (0 < M <= 1 << 20 and L.bit_length() + M.bit_length() <= 31 and values is not None
                and _fits(ids, _I64, index, shape) and _fits(values, _F32, index, shape)):
            return None
        bias_stride = M if ids.dim() == 2 else 0
    elif values is not None:
        return None
    if mask is not None:
        S = mask.shape[0] if mask.dim() else 0
        if not (S and _fits(mask, torch.int32, index, (S, (V + 31) // 32))
                and (S in (1, B) if state is None else _fits(state, _I64, index, row))):
            return None
    elif state is not None:
        return None
    got = logits.new_empty(B, dtype=_I64) if choose else torch.empty_like(logits)
    nbytes = _gen_workspace(B, V) if choose else 0
    ws = logits.new_empty(nbytes, dtype=torch.uint8) if nbytes else None
    at = got.data_ptr()
    rc = gen_lib().pragnosia_rules(logits.data_ptr(), dt is _BF16, _at(history), stride, L, _at(lengths), _at(prompt),
                                   *args, _at(ids), _at(values), M, bias_stride, _at(mask), S, _at(state),
                                   None if choose else at, at if choose else None, _at(ws), nbytes, B, V,
                                   _raw_stream(index))
    if rc:
        check(rc, "pragnosia_rules")
    return got


def _run(logits, history, lengths, prompt, penalties, ids, values, mask, state, choose: bool) -> Tensor:
    logits = _as(logits, logits.dtype)
    got = logits.new_empty(logits.shape[0], dtype=_I64) if choose else torch.empty_like(logits)
    _launch(logits, history, lengths, prompt, penalties, ids, values, mask, state, None if choose else got,
            got if choose else None)
    return got


def apply_rules(logits: Tensor, history: Optional[Tensor] = None, lengths: Optional[Tensor] = None,
                prompt: Optional[Tensor] = None, *, repetition: Penalty = 1.0, presence: Penalty = 0.0,
                frequency: Penalty = 0.0, bias: Optional[tuple[Tensor, Tensor]] = None, mask: Optional[Tensor] = None,
                state: Optional[Tensor] = None) -> Tensor:
    """logits (B, V), fp32 or bf16, under the rules above, in a new tensor of their type (rounded once).

    history (B, L): each row's token ids, of which the first lengths[b] (all by default) are there and those from
    prompt[b] (0 by default) on were generated; ids outside [0, V) take no part, lengths and prompt are clamped to
    [0, L]. repetition (above 0), presence and frequency: a number finite in fp32, or a (B,) tensor for each row its own, whose
    values are taken as they are. bias: (ids,
    values), both (M) or (B, M): the last entry of a repeated id counts, ids outside [0, V) are skipped, -inf bans a
    word whose logit is finite (of an infinity or a NaN it makes a NaN; a mask bans any); L and M must have 31 bits together
    at most (2^15 entries on 2^15 tokens). mask (S, ceil(V / 32)) int32: word v is allowed where bit v % 32 of word v // 32 is
    set; state (B) picks each row's line (by default its own of B, or the only one): a negative state leaves the row
    unmasked, one of S or more masks every word. For inference: no input may require a gradient where gradients are
    recorded."""
    return _rules("apply_rules", logits, history, lengths, prompt, repetition, presence, frequency, bias, mask, state,
                  False)


def next_token(logits: Tensor, history: Optional[Tensor] = None, lengths: Optional[Tensor] = None,
               prompt: Optional[Tensor] = None, *, repetition: Penalty = 1.0, presence: Penalty = 0.0,
               frequency: Penalty = 0.0, bias: Optional[tuple[Tensor, Tensor]] = None, mask: Optional[Tensor] = None,
               state: Optional[Tensor] = None) -> Tensor:
    """The word of each row's largest logit under the rules (`apply_rules`), (B,) int64: the lowest among equals, NaN
    above every number as in torch.argmax; -1 where nothing is left (every word masked, banned or at -inf). The fp32 values
    are compared, also of bf16 logits."""
    return _rules("next_token", logits, history, lengths, prompt, repetition, presence, frequency, bias, mask, state, True)


def advance(tokens: Tensor, history: Optional[Tensor] = None, lengths: Optional[Tensor] = None,
            next: Optional[Tensor] = None, state: Optional[Tensor] = None, *, vocab: Optional[int] = None) -> None:
    """What follows a chosen token, in place and without the host: history[b, lengths[b]] = tokens[b] and lengths[b] one
    more (while there is room), state[b] = next[state[b], tokens[b]] (for a state in [0, S)). tokens, lengths and state (B)
    and history (B, L) int64, next (S, V) int32; history with lengths, next with state, either pair or both. Rows whose token
    is outside the vocabulary (-1: nothing was left) stay as they are; without next, the vocabulary is `vocab` words."""
    if next is None and vocab is None:
        raise PragnosiaError("advance: the vocabulary's size, as `next` or `vocab`, is needed")
    V = vocab if next is None else next.shape[-1] if next.dim() else 0
    _check_advance("advance", tokens, history, lengths, next, state, V)
    if _watched(tokens, history, lengths, next, state):
        raise PragnosiaError("advance: not available in a trace or under a dispatch mode (it works in place)")
    _tail(tokens, history, lengths, next, state, V)


def _check_advance(op: str, tokens, history, lengths, next, state, V: int) -> None:
    _require_gpu(tokens, history, lengths, next, state)
    if (history is None) != (lengths is None) or (next is None) != (state is None) or (history is None and next is None):
        raise PragnosiaError(f"{op}: history with lengths, next with state, either pair or both expected")
    B = tokens.numel()
    _expect(op, tokens.device, tokens=(tokens, (B,)), history=(history, (B, None)), lengths=(lengths, (B,)),
            next=(next, (None, V)), state=(state, (B,)))
    for name, t in (("tokens", tokens), ("history", history), ("lengths", lengths), ("state", state)):
        if t is not None and (t.dtype != _I64 or not (t.is_contiguous() or (name == "history" and t.stride(1) == 1 and
                                                                            t.stride(0) >= t.shape[1]))):
            raise PragnosiaError(f"{op}: {name} must be int64 and dense (history's rows), as it is changed in place")
    if next is not None and (next.dtype != torch.int32 or not next.is_contiguous() or next.numel() == 0):
        raise PragnosiaError(f"{op}: next (S, V) must be dense int32 with S > 0 and V > 0, got {tuple(next.shape)} "
                             f"{next.dtype}")
    if history is not None and history.shape[1] == 0:
        raise PragnosiaError(f"{op}: a history of no entries has no room")


def _tail(tokens, history, lengths, next, state, V: int, step=None) -> None:
    """The C call. step: the rest of a decode step as decode.GreedyDecoder keeps it, or None."""
    B = tokens.shape[0]
    if B == 0:
        return
    emb = [None, None, 0, 0] + [None] * 5 + [0, None, None, None, 0]
    if step is not None:
        e, pe, ctr_in, ctr_out, pos_in, pos_out, out, tok, h, p0s = step
        if not (all(t.dtype == _F32 and t.is_contiguous() for t in (e, pe, h, p0s)) and e.shape == (V, h.shape[1])
                and pe.shape[1] == e.shape[1] and h.shape[0] == B and out.shape[1] == B and tok.numel() == B):
            raise PragnosiaError("advance: the step's buffers do not have the decoder's shapes and types")
        emb = [_at(e), _at(pe), e.shape[1], pe.shape[0], _at(ctr_in), _at(ctr_out), _at(pos_in), _at(pos_out), _at(out),
               out.shape[0], _at(tok), _at(h), _at(p0s), p0s.numel()]
    _call("pragnosia_rules_tail", gen_lib().pragnosia_rules_tail, tokens, _at(tokens), _at(history),
          0 if history is None else history.stride(0), 0 if history is None else history.shape[1], _at(lengths), _at(next),
          0 if next is None else next.shape[0], _at(state), *emb, B, V)


@dataclasses.dataclass
class TokenRules:
    """Rules that `GreedyDecoder` chooses tokens under, with the meanings of `next_token`: repetition counts the prompt,
    presence and frequency what was generated. A grammar is an automaton on the GPU: `mask` (S, ceil(V / 32)) holds the words
    allowed in each state, `next` (S, V) int32 the state after each word (-1: free from then on; S or more: nothing may
    follow), `state` (B) the states to begin in (0 by default, for every sequence). Without `next` the states stay."""
    repetition: Penalty = 1.0
    presence: Penalty = 0.0
    frequency: Penalty = 0.0
    bias: Optional[tuple[Tensor, Tensor]] = None
    mask: Optional[Tensor] = None
    state: Optional[Tensor] = None
    next: Optional[Tensor] = None


class RuleState:
    """TokenRules, and the history and states of B sequences they are applied to, in buffers that a captured graph reads."""

    def __init__(self, rules: TokenRules, B: int, V: int, capacity: int, device):
        self.B, self.V, self.capacity = B, V, capacity
        self.shapes = self.shapes_of(rules)
        e = lambda *s, dt=_I64: torch.zeros(*s, device=device, dtype=dt)  # noqa: E731
        self.history, self.lengths, self.prompt = e(B, capacity), e(B), e(B)
        self.penalties = [e(B, dt=_F32) for _ in range(3)]
        ids, _, mask, _, nxt = self.shapes
        self.bias = None if ids is None else (e(*ids), e(*ids, dt=_F32))
        self.mask = None if mask is None else e(*mask, dt=torch.int32)
        self.next = None if nxt is None else e(*nxt, dt=torch.int32)
        self.state = e(B) if mask is not None else None  # (0, also of a mask that has as many lines as there are rows)

    @staticmethod
    def shapes_of(rules: TokenRules):
        ids, values = (None, None) if rules.bias is None else rules.bias
        return tuple(None if t is None else tuple(t.shape) for t in (ids, values, rules.mask, rules.state, rules.next))

    @staticmethod
    def check(rules: TokenRules, prompt: Optional[Tensor], B: int, V: int, capacity: int) -> None:
        """Refuses what `load` or a step would not take, before anything is made or written. A tensor of one value for B
        counts for every sequence."""
        def no(what, got):
            raise PragnosiaError(f"TokenRules: {what} expected, got {got}")

        def shown(t):
            return f"{tuple(t.shape)} {t.dtype}"

        each = ((B,), (1,), ())
        if capacity > 1 << 24:
            no("a prompt and a run of at most 2^24 tokens together", capacity)
        if prompt is not None and (prompt.dim() != 2 or prompt.shape[0] not in (1, B) or prompt.dtype not in _INTS):
            no(f"a prompt of integers ({B}, P)", shown(prompt))
        for name in ("repetition", "presence", "frequency"):
            p = getattr(rules, name)
            if isinstance(p, Tensor):
                if tuple(p.shape) not in each or not (p.is_floating_point() or p.dtype in _INTS):
                    no(f"{name}, a number or numbers ({B},),", shown(p))
            elif not _in_range(name, p):
                raise _out_of_range("TokenRules", name, p)
        if rules.bias is not None:
            ids, values = rules.bias
            if (ids.dim() not in (1, 2) or (ids.dim() == 2 and ids.shape[0] != B) or ids.shape[-1] > 1 << 20
                    or ids.dtype not in _INTS):
                no(f"bias ids, integers (M) or ({B}, M) with M up to 2^20,", shown(ids))
            if values.shape != ids.shape or not (values.is_floating_point() or values.dtype in _INTS):
                no(f"bias values {tuple(ids.shape)}", shown(values))
            if not _marks_fit(capacity, ids.shape[-1]):
                no("prompt, run and bias list of 31 bits together at most", (capacity, ids.shape[-1]))
        mask, state, nxt, words = rules.mask, rules.state, rules.next, (V + 31) // 32
        if mask is not None and (mask.dim() != 2 or mask.shape[0] == 0 or mask.shape[1] != words
                                 or mask.dtype not in (torch.int32, _I64)):
            no(f"mask (S, {words}) int32 with S > 0", shown(mask))
        if state is not None and (mask is None or tuple(state.shape) not in each or state.dtype not in _INTS):
            no(f"state, integers ({B},) beside a mask,", shown(state))
        if nxt is not None and (mask is None or tuple(nxt.shape) != (mask.shape[0], V)
                                or nxt.dtype not in _INTS):
            no("next (S, V) int32 beside mask (S, words)", shown(nxt))

    def load(self, rules: TokenRules, prompt: Optional[Tensor]) -> None:
        """The rules' present values, the prompt (B, P) as history, and the states to begin in; all checked before."""
        for name, buf in zip(("repetition", "presence", "frequency"), self.penalties):
            p = getattr(rules, name)
            buf.copy_(p) if isinstance(p, Tensor) else buf.fill_(float(p))
        if self.bias is not None:
            self.bias[0].copy_(rules.bias[0]), self.bias[1].copy_(rules.bias[1])
        if self.mask is not None:
            self.mask.copy_(rules.mask)
        if self.next is not None:
            nxt = rules.next  # (64-bit states past 32 bits stay past the last)
            self.next.copy_(nxt.clamp(-1, nxt.shape[0]) if nxt.dtype == _I64 else nxt)
        if self.state is not None:
            self.state.zero_() if rules.state is None else self.state.copy_(rules.state)
        P = 0 if prompt is None else prompt.shape[1]
        if P:
            self.history[:, :P].copy_(prompt)
        self.lengths.fill_(P)
        self.prompt.fill_(P)

    def choose(self, logits: Tensor) -> Tensor:
        r, p, f = self.penalties
        return next_token(logits, self.history, self.lengths, self.prompt, repetition=r, presence=p, frequency=f,
                          bias=self.bias, mask=self.mask, state=self.state)

    def advance(self, tokens: Tensor, step=None) -> None:
        state = self.state if self.next is not None else None
        _check_advance("advance", tokens, self.history, self.lengths, self.next, state, self.V)
        _tail(tokens, self.history, self.lengths, self.next, state, self.V, step)


# ---------------------------------------------------------------------------------------------------------------
# the same as custom ops, for traces
def _op(op: str, choose: bool, logits, history, lengths, prompt, tensors, numbers, ids, values, mask, state):
    penalties = tuple(n if t is None else t for t, n in zip(tensors, numbers))
    _checked(op, logits, history, lengths, prompt, tuple(zip(("repetition", "presence", "frequency"), penalties)), ids,
             values, mask, state)
    _no_tangents(op, logits, values, *tensors)
    return _run(logits, history, lengths, prompt, penalties, ids, values, mask, state, choose)


@torch.library.custom_op("pragnosia_gen::rules_apply", mutates_args=())
def rules_apply(logits: Tensor, history: Optional[Tensor], lengths: Optional[Tensor], prompt: Optional[Tensor],
                repetition: Optional[Tensor], repetition_value: float, presence: Optional[Tensor], presence_value: float,
                frequency: Optional[Tensor], frequency_value: float, bias_ids: Optional[Tensor],
                bias_values: Optional[Tensor], mask: Optional[Tensor], state: Optional[Tensor]) -> Tensor:
    """The logits under the rules; a penalty's number counts where its tensor is None."""
    return _op("rules_apply", False, logits, history, lengths, prompt, (repetition, presence, frequency),
               (repetition_value, presence_value, frequency_value), bias_ids, bias_values, mask, state)


@rules_apply.register_fake
def _(logits, *rest):
    return torch.empty_like(logits, memory_format=torch.contiguous_format)


@torch.library.custom_op("pragnosia_gen::rules_token", mutates_args=())
def rules_token(logits: Tensor, history: Optional[Tensor], lengths: Optional[Tensor], prompt: Optional[Tensor],
                repetition: Optional[Tensor], repetition_value: float, presence: Optional[Tensor], presence_value: float,
                frequency: Optional[Tensor], frequency_value: float, bias_ids: Optional[Tensor],
                bias_values: Optional[Tensor], mask: Optional[Tensor], state: Optional[Tensor]) -> Tensor:
    """The token that the rules leave, -1 where there is none."""
    return _op("rules_token", True, logits, history, lengths, prompt, (repetition, presence, frequency),
               (repetition_value, presence_value, frequency_value), bias_ids, bias_values, mask, state)


@rules_token.register_fake
def _(logits, *rest):
    return logits.new_empty(logits.shape[0], dtype=_I64)
