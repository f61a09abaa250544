"""Rules for the next token, on hand-written kernels (csrc/rules.hip; C ABI in pragnosia_amd/include/pragnosia_gen.h): penalties
for repeated tokens, biases of some words, masks of what a grammar allows, in one pass over the logits.

    token = next_token(logits, history, lengths, prompt, repetition=1.2, bias=(ids, values), mask=mask, state=state)
    logits = apply_rules(logits, ...)           # the same rules, the logits for a sampler of the caller's own

For row b and word v, in fp32, each step rounded:

    a word among history[b, :lengths[b]]                x = l / repetition where l > 0, else l * repetition
    c > 0 times among history[b, prompt[b]:lengths[b]]  x = x - presence, then x = x - frequency * c
    a word of the row's bias list                       x = x + its value
    a word whose mask bit is clear                      x = -inf

`GreedyDecoder(..., rules=TokenRules(...))` chooses its tokens under them; the reference takes the argmax or samples the
logits as they are (`src/bench.py:83`).
"""
from __future__ import annotations

import math
from typing import Optional, Union

import torch
from torch import Tensor

from ._lib import PragnosiaError, check, gen_lib
from .fp4 import _device, _fits, _quiet
from .head import _BF16, _F32, _FLOATS, _I64, _INTS, _as, _at, _call, _no_tangents, _raw_stream, _watched
from .ops import _expect, _require_gpu

Penalty = Union[float, Tensor]


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
        elif not math.isfinite(p) or (name == "repetition" and p <= 0):
            raise PragnosiaError(f"{op}: {name} must be finite{' and above 0' if name == 'repetition' else ''}, got {p}")
    if (ids is None) != (values is None):
        raise PragnosiaError(f"{op}: bias is (ids, values)")
    if ids is not None:
        if ids.dim() not in (1, 2) or (ids.dim() == 2 and ids.shape[0] != B) or ids.shape[-1] > 1 << 20:
            raise PragnosiaError(f"{op}: bias ids (M) or ({B}, M) with M up to 2^20 expected, got {tuple(ids.shape)}")
        _expect(op, dev, bias_ids=(ids, tuple(ids.shape)), bias_values=(values, tuple(ids.shape)))
        if history is not None and history.shape[1].bit_length() + ids.shape[-1].bit_length() > 31:
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
    if logits.dim() != 2:
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
    if not (isinstance(args[1], float) and 0.0 < args[1] < math.inf and math.isfinite(args[3]) and math.isfinite(args[5])):
        return None
    if ids is not None:
        M = ids.shape[-1]
        shape = row + (M,) if ids.dim() == 2 else (M,)
        if not (0 < M <= 1 << 20 and L.bit_length() + M.bit_length() <= 31 and values is not None and _fits(ids, _I64, index, shape) and _fits(values, _F32, index, shape)):
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
    if not _quiet({type(t) for t in (logits, history, lengths, prompt, *penalties, ids, values, mask, state)}):
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
    [0, L]. repetition (above 0), presence and frequency: a number, or a (B,) tensor for each row its own. bias: (ids,
    values), both (M) or (B, M): the last entry of a repeated id counts, ids outside [0, V) are skipped, -inf bans a
    word; L and M must have 31 bits together at most (2^15 entries on 2^15 tokens). mask (S, ceil(V / 32)) int32: word v is allowed where bit v % 32 of word v // 32 is set; state (B) picks each
    row's line (by default its own of B, or the only one): a negative state leaves the row unmasked, one of S or more
    masks every word. For inference: no input may require a gradient where gradients are recorded."""
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
