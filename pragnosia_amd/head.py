"""The head's losses over the vocabulary, with no logits kept: cross entropy of labels and distillation from a teacher's
top logits, forward and backward on hand-written kernels (csrc/head_loss.hip; C ABI in
pragnosia_amd/include/pragnosia_lm.h).

    loss, lse = linear_cross_entropy(h, W, y)
    kd, ce = linear_distill(h, W, ids, logits, tau, y)

h (..., d) are hidden rows and W (V, d) the head's weight (the LM's tied table), d a multiple of 8. The logits h W^T are
formed on the bf16 matrix cores in pieces of the vocabulary: fp32 h and W are rounded to bf16, as autocast rounds a
Linear's operands. The reference's LM forms its logits in chunks of rows under activation checkpointing
(`src/model.py:563-567`); LM.loss does so here too, unless the model was built with fused_ends.

Every loss comes per token in fp32, so a mean, a mask or weights are the caller's own: the kernels take the per-token
gradients that autograd hands back. The gradients of logits are rounded to bf16 once, before the two products that dh
(in h's type, but always rounded to bf16 first, as autocast's product gives it) and dW (in W's; an fp32 W gets the
unrounded fp32 sums) are; sums are held in fp32 throughout and taken in a fixed order, so the same call gives the same
bits.

An eager call goes through an autograd function straight to the C ABI. One that something records or replaces
(torch.compile, torch.export, make_fx, torch.jit.trace, a dispatch mode, tensors of another class) goes through the
custom ops, whose dispatch costs tens of microseconds a call. Derivatives are reverse mode, once: forward-mode tangents,
second derivatives and torch.func's transforms raise.
"""
from __future__ import annotations

import functools
import math
from typing import Optional

import torch
from torch import Tensor
from torch.autograd import forward_ad

from ._lib import PragnosiaError, check, lm_lib
from .ops import _expect, _require_gpu

_FLOATS = (torch.bfloat16, torch.float32)
_INTS = (torch.int64, torch.int32, torch.int16, torch.int8, torch.uint8)
_F32, _BF16, _I64 = torch.float32, torch.bfloat16, torch.int64
_TAU = (2.0 ** -10, 2.0 ** 10)  # past these tau^2 kd or the scaled logits' rounding leaves little of an fp32 loss


def _as(t: Optional[Tensor], dtype: torch.dtype) -> Optional[Tensor]:
    """t in `dtype`, contiguous, at an address the kernels' 16-byte loads take (a slice may start anywhere)."""
    if t is None:
        return None
    if t.dtype != dtype or not t.is_contiguous():
        t = t.to(dtype).contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _at(t: Optional[Tensor]):
    return None if t is None else t.data_ptr()


_raw_stream = torch._C._cuda_getCurrentRawStream  # current_stream(i).cuda_stream without the Python object


def _call(what: str, fn, t: Tensor, *args) -> None:
    """fn(*args, the current stream of t's device), with that device the current one."""
    index = t.device.index
    if index == torch.cuda.current_device():
        rc = fn(*args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            rc = fn(*args, _raw_stream(index))
    if rc:
        check(rc, what)


_Parameter, _compiling, _modes = torch.nn.Parameter, torch.compiler.is_compiling, torch._C._len_torch_dispatch_stack
_tracing, _included = torch._C._is_tracing, torch._C._dispatch_tls_is_dispatch_key_included
_PRE = torch._C.DispatchKey.PreDispatch


def _watched(*ts: Optional[Tensor]) -> bool:
    """Whether torch's operations on these tensors are recorded or replaced by something other than autograd: a trace, a
    dispatch mode, a tensor class of its own. The direct calls are no operations to it; the custom ops are."""
    if _compiling() or _modes() or _tracing() or _included(_PRE):
        return True
    for t in ts:
        if t is not None and type(t) is not Tensor and type(t) is not _Parameter:
            return True
    return False


def _no_tangents(op: str, *ts: Optional[Tensor]) -> None:
    """A tensor with a forward-mode tangent is refused: the kernels have no forward derivative, and the result would go
    on without one."""
    if forward_ad._current_level >= 0 and any(t is not None and forward_ad.unpack_dual(t).tangent is not None
                                              for t in ts):
        raise PragnosiaError(f"{op}: forward-mode derivatives are not available (use reverse mode)")


def _once(backward):
    """A backward whose results cannot be differentiated again: refused (once_differentiable, whose wrapper costs as
    much as a short call's launches) where a graph of the backward is built, direct otherwise."""
    refusing = torch.autograd.function.once_differentiable(backward)

    def run(ctx, *grads):
        return (refusing if torch.is_grad_enabled() else backward)(ctx, *grads)

    return run


@functools.lru_cache(maxsize=4096)
def _workspace(what: str, *sizes: int) -> int:
    """A workspace query of the C ABI: a function of the sizes alone."""
    nbytes = getattr(lm_lib(), what)(*sizes)
    if nbytes < 0:
        raise PragnosiaError(f"{what}: sizes {sizes} rejected")
    return nbytes


def _plain_call(h: Tensor, W: Tensor, y: Optional[Tensor], ids: Optional[Tensor], z: Optional[Tensor],
                tau: float) -> bool:
    """Whether _check_head has nothing to say, at a fraction of its cost on the host."""
    if not (h.is_cuda and h.dim() == 2 and W.dim() == 2 and h.dtype in _FLOATS and W.dtype in _FLOATS):
        return False
    (n, d), dev = h.shape, h.device
    if not (W.device == dev and W.shape[1] == d and W.shape[0] > 0 and d > 0 and d % 8 == 0):
        return False
    if y is not None and not (y.device == dev and y.dtype is _I64 and y.dim() == 1 and y.shape[0] == n):
        return False
    if ids is None:
        return y is not None and z is None
    return (z is not None and ids.device == dev and z.device == dev and ids.dtype is _I64 and z.dtype is _F32
            and ids.dim() == 2 and ids.shape[0] == n and 0 < ids.shape[1] <= 1024 and z.shape == ids.shape
            and _TAU[0] <= tau <= _TAU[1])


def _check_head(op: str, h: Tensor, W: Tensor, y: Optional[Tensor], ids: Optional[Tensor], z: Optional[Tensor],
                tau: float) -> None:
    _require_gpu(h, W, y, ids, z)
    if h.dim() != 2 or W.dim() != 2:
        raise PragnosiaError(f"{op}: h (..., d) and W (V, d) expected, got {tuple(h.shape)} and {tuple(W.shape)}")
    n, d = h.shape
    _expect(op, h.device, W=(W, (None, d)), y=(y, (n,)), ids=(ids, (n, None)))
    if h.dtype not in _FLOATS or W.dtype not in _FLOATS:
        raise PragnosiaError(f"{op}: h and W must be bf16 or fp32, got {h.dtype} and {W.dtype}")
    if d == 0 or d % 8 or W.shape[0] == 0:
        raise PragnosiaError(f"{op}: the width must be a multiple of 8 and the vocabulary not empty, got W "
                             f"{tuple(W.shape)}")
    for name, t in (("y", y), ("ids", ids)):
        if t is not None and t.dtype not in _INTS:
            raise PragnosiaError(f"{op}: {name} must be integers, got {t.dtype}")
    if (ids is None) != (z is None) or (y is None and ids is None):
        raise PragnosiaError(f"{op}: labels, or a teacher's ids and logits together, expected")
    if ids is not None:
        _expect(op, h.device, logits=(z, tuple(ids.shape)))
        if not 0 < ids.shape[1] <= 1024 or not z.is_floating_point():
            raise PragnosiaError(f"{op}: ids and logits (..., K) with K from 1 to 1024 and floating logits expected, "
                                 f"got {tuple(ids.shape)} and {z.dtype}")
    if not _TAU[0] <= tau <= _TAU[1]:
        raise PragnosiaError(f"{op}: tau must be from {_TAU[0]} to {_TAU[1]}, got {tau}")


def _forward(h: Tensor, W: Tensor, y: Optional[Tensor], ids: Optional[Tensor], z: Optional[Tensor], tau: float):
    """h (n, d), W (V, d) bf16; y (n) int64 or None; ids int64 and z fp32 (n, K) or None, all contiguous. Returns (ce,
    lse, kd, stats): fp32, None where not asked for; stats (int32: bits) holds lse_t, psum, entry, p and zl for the
    backward."""
    n, d = h.shape
    V, K = W.shape[0], 0 if ids is None else ids.shape[1]
    e = lambda s: torch.empty(s, device=h.device, dtype=_F32)
    ce, lse = (None, None) if y is None else (e(n), e(n))
    kd, stats = (None, None) if ids is None else (e(n), e(n * (2 + 3 * K)).view(torch.int32))
    if n == 0:
        return ce, lse, kd, stats
    nbytes = _workspace("pragnosia_head_fwd_workspace_bytes", n, V, d, K)
    ws = torch.empty(nbytes, device=h.device, dtype=torch.uint8)
    _call("pragnosia_head_fwd", lm_lib().pragnosia_head_fwd, h, _at(h), _at(W), _at(y), _at(ids), _at(z), tau, _at(ce),
          _at(lse), _at(kd), *_stats_at(stats, n, K), _at(ws), nbytes, n, V, d, K)
    return ce, lse, kd, stats


def _stats_at(stats: Optional[Tensor], n: int, K: int):
    """Addresses of lse_t, psum, entry, p, zl in `stats`."""
    if stats is None:
        return (None,) * 5
    a = stats.data_ptr()
    return a, a + 4 * n, a + 8 * n, a + 8 * n + 4 * n * K, a + 8 * n + 8 * n * K


def _backward(g_ce, g_lse, g_kd, h, W, y, lse, stats, K: int, tau: float, need_h: bool, need_W: bool, dw_f32: bool):
    """Gradients of ce, lse and kd ((n,) or None) -> (dh bf16, dW bf16 or fp32), None where not needed."""
    n, d = h.shape
    V = W.shape[0]
    dW_type = _F32 if dw_f32 else _BF16
    if n == 0 or (g_ce is None and g_lse is None and g_kd is None):
        return (h.new_zeros(n, d) if need_h else None,
                W.new_zeros(V, d, dtype=dW_type) if need_W else None)
    dh = torch.empty_like(h) if need_h else None
    dW = torch.empty(V, d, device=h.device, dtype=dW_type) if need_W else None
    g_ce, g_lse, g_kd = _as(g_ce, _F32), _as(g_lse, _F32), _as(g_kd, _F32)
    nbytes = _workspace("pragnosia_head_bwd_workspace_bytes", n, V, d)
    ws = torch.empty(nbytes, device=h.device, dtype=torch.uint8)
    _call("pragnosia_head_bwd", lm_lib().pragnosia_head_bwd, h, _at(g_ce), _at(g_lse), _at(g_kd), _at(h), _at(W),
          _at(y), _at(lse), *_stats_at(stats, n, K), tau, _at(dh), _at(dW), dw_f32, _at(ws), nbytes, n, V, d, K)
    return dh, dW


def _operands(h, W, y, ids, z):
    return _as(h, _BF16), _as(W, _BF16), _as(y, _I64), _as(ids, _I64), _as(z, _F32)


class _HeadLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, h, W, y, ids, z, tau):
        h16, W16, y, ids, z = _operands(h, W, y, ids, z)
        ce, lse, kd, stats = _forward(h16, W16, y, ids, z, tau)
        ctx.save_for_backward(h16, W16, y, lse, stats)
        ctx.tau, ctx.K, ctx.types = tau, 0 if ids is None else ids.shape[1], (h.dtype, W.dtype)
        ctx.set_materialize_grads(False)  # an unused output's gradient arrives as None, not zeros
        return ce, lse, kd

    @staticmethod
    @_once
    def backward(ctx, g_ce, g_lse, g_kd):
        _no_tangents("head_loss_bwd", g_ce, g_lse, g_kd)
        h, W, y, lse, stats = ctx.saved_tensors
        need_h, need_W = ctx.needs_input_grad[:2]
        if _watched(g_ce, g_lse, g_kd):
            none = W.new_empty(0, dtype=_F32)
            dh, dW = head_loss_bwd(g_ce, g_lse, g_kd, h.to(ctx.types[0]), W.to(ctx.types[1]), y,
                                   none if lse is None else lse, none.to(torch.int32) if stats is None else stats,
                                   ctx.tau, need_h, need_W)
            return dh if need_h else None, dW if need_W else None, None, None, None, None
        dh, dW = _backward(g_ce, g_lse, g_kd, h, W, y, lse, stats, ctx.K, ctx.tau, need_h, need_W,
                           ctx.types[1] == _F32)
        if dh is not None and ctx.types[0] != _BF16:
            dh = dh.to(ctx.types[0])
        return dh, dW, None, None, None, None


# ---------------------------------------------------------------------------------------------------------------
# the same as custom ops, for traces
@torch.library.custom_op("pragnosia_lm::head_loss", mutates_args=())
def head_loss(h: Tensor, W: Tensor, y: Optional[Tensor], ids: Optional[Tensor], z: Optional[Tensor],
              tau: float) -> tuple[Tensor, Tensor, Tensor, Tensor]:
    """h (n, d), W (V, d), y (n) or None, ids and z (n, K) or None. Returns (ce, lse, kd, stats), empty where there are
    no labels or no teacher; stats is what the backward takes."""
    _check_head("head_loss", h, W, y, ids, z, tau)
    _no_tangents("head_loss", h, W)
    got = _forward(*_operands(h, W, y, ids, z), float(tau))
    types = (_F32, _F32, _F32, torch.int32)
    return tuple(t if t is not None else torch.empty(0, device=h.device, dtype=dt) for t, dt in zip(got, types))


@head_loss.register_fake
def _(h, W, y, ids, z, tau):
    n, K = h.shape[0], 0 if ids is None else ids.shape[1]
    e = lambda s: h.new_empty(s, dtype=_F32)
    ny, nk = (0 if y is None else n), (0 if ids is None else n)
    return e(ny), e(ny), e(nk), h.new_empty(nk * (2 + 3 * K), dtype=torch.int32)


@torch.library.custom_op("pragnosia_lm::head_loss_bwd", mutates_args=())
def head_loss_bwd(g_ce: Optional[Tensor], g_lse: Optional[Tensor], g_kd: Optional[Tensor], h: Tensor, W: Tensor,
                  y: Optional[Tensor], lse: Tensor, stats: Tensor, tau: float, need_h: bool,
                  need_W: bool) -> tuple[Tensor, Tensor]:
    """Gradients of head_loss's ce, lse and kd -> (dh, dW) in h's and W's types; empty where not needed. y as given to
    head_loss, lse and stats as it returned them."""
    _require_gpu(g_ce, g_lse, g_kd, h, W, y, lse, stats)
    _no_tangents("head_loss_bwd", g_ce, g_lse, g_kd, h, W)
    if h.dim() != 2 or W.dim() != 2 or h.dtype not in _FLOATS or W.dtype not in _FLOATS:
        raise PragnosiaError(f"head_loss_bwd: h (n, d) and W (V, d) expected, got {tuple(h.shape)}, {tuple(W.shape)}")
    n, d = h.shape
    _expect("head_loss_bwd", h.device, W=(W, (None, d)), g_ce=(g_ce, (n,)), g_lse=(g_lse, (n,)), g_kd=(g_kd, (n,)),
            y=(y, (n,)), lse=(lse if y is not None else None, (n,)), stats=(stats, (None,)))
    K = (stats.numel() // n - 2) // 3 if n and stats.numel() else 0
    if stats.numel() not in (0, n * (2 + 3 * K)) or lse.dtype != _F32 or stats.dtype != torch.int32:
        raise PragnosiaError("head_loss_bwd: lse and stats must be head_loss's")
    # (of no tokens there are no entries to tell K by, and the gradients are zeros)
    if (y is None and (g_ce is not None or g_lse is not None)) or (n and K == 0 and g_kd is not None):
        raise PragnosiaError("head_loss_bwd: a gradient of a loss that was not computed")
    dh, dW = _backward(g_ce, g_lse, g_kd, _as(h, _BF16), _as(W, _BF16), _as(y, _I64),
                       None if y is None else _as(lse, _F32), _as(stats, torch.int32) if K else None, K, float(tau),
                       need_h, need_W, W.dtype == _F32)
    return (h.new_empty(0, d) if dh is None else dh.to(h.dtype)), (W.new_empty(0, d) if dW is None else dW)


@head_loss_bwd.register_fake
def _(g_ce, g_lse, g_kd, h, W, y, lse, stats, tau, need_h, need_W):
    n, d = h.shape
    return h.new_empty(n if need_h else 0, d), W.new_empty(W.shape[0] if need_W else 0, d)


def _head_setup(ctx, inputs, output):
    ctx.set_materialize_grads(False)
    h, W, y, ids, z, tau = inputs
    _, lse, _, stats = output
    ctx.tau, ctx.has = tau, (y is not None, ids is not None)
    ctx.save_for_backward(h, W, y, lse, stats)
    ctx.mark_non_differentiable(stats)


def _head_backward(ctx, g_ce, g_lse, g_kd, _):
    h, W, y, lse, stats = ctx.saved_tensors
    need_h, need_W = ctx.needs_input_grad[:2]
    has_y, has_kd = ctx.has
    dh, dW = head_loss_bwd(g_ce if has_y else None, g_lse if has_y else None, g_kd if has_kd else None, h, W, y, lse,
                           stats, ctx.tau, need_h, need_W)
    return dh if need_h else None, dW if need_W else None, None, None, None, None


head_loss.register_autograd(_head_backward, setup_context=_head_setup)


def _losses(op: str, h: Tensor, W: Tensor, y: Optional[Tensor], ids: Optional[Tensor], z: Optional[Tensor],
            tau: float):
    """(ce, lse, kd) in h's leading shape."""
    lead = h.shape[:-1]
    if h.dim() < 1 or (y is not None and y.shape != lead) or any(
            t is not None and (t.dim() != h.dim() or t.shape[:-1] != lead) for t in (ids, z)):
        raise PragnosiaError(f"{op}: the labels' and the teacher's leading sizes must be h's {tuple(lead)}, got "
                             f"{[None if t is None else tuple(t.shape) for t in (y, ids, z)]}")
    _no_tangents(op, h, W)
    flat = h.dim() == 2
    if not flat:
        h = h.reshape(-1, h.shape[-1])
        y = None if y is None else y.reshape(-1)
        ids, z = (None, None) if ids is None else (ids.reshape(-1, ids.shape[-1]), z.reshape(-1, z.shape[-1]))
    if _watched(h, W, y, ids, z):
        got = head_loss(h, W, y, ids, z, tau)[:3]
    else:
        if not _plain_call(h, W, y, ids, z, tau):
            _check_head(op, h, W, y, ids, z, tau)
        if torch.is_grad_enabled() and (h.requires_grad or W.requires_grad):
            got = _HeadLoss.apply(h, W, y, ids, z, tau)
        else:
            got = _forward(*_operands(h, W, y, ids, z), tau)[:3]
    return got if flat else tuple(t if t is None else t.view(lead) if t.numel() or 0 in lead else t for t in got)


def linear_cross_entropy(h: Tensor, W: Tensor, y: Tensor) -> tuple[Tensor, Tensor]:
    """Per-token cross entropy of the head h W^T at the labels y, and the log of the softmax's denominator (for a
    penalty on it, or a label's log-probability elsewhere): both y's shape, fp32, both differentiable in h and W.

    A label outside [0, V) (padding, such as -100) has loss 0 and adds no gradient. Such rows of h still enter dW's
    sums, times zero: they have to be finite there."""
    return _losses("linear_cross_entropy", h, W, y, None, None, 1.0)[:2]


def linear_distill(h: Tensor, W: Tensor, ids: Tensor, logits: Tensor, tau: float = 1.0,
                   y: Optional[Tensor] = None) -> tuple[Tensor, Optional[Tensor]]:
    """Per-token distillation loss of the head h W^T from a teacher's top logits, and with labels y the cross entropy
    (else None) from the same pass over the vocabulary; fp32, h's leading shape, differentiable in h and W.

    ids and logits (..., K), K up to 1024: the teacher's words, in any order, and its logits there. Its distribution p
    is their softmax at temperature tau (2^-10 to 2^10); the loss is tau^2 KL(p || q) with q the softmax of the
    student's logits over the whole vocabulary at tau. An id outside [0, V) marks an entry that is not there (lists of
    different lengths), whatever its logit; a logit of -inf has probability zero; a token with no entry left has loss 0
    and no gradient; a NaN among a token's logits makes its loss NaN. A repeated id has the sum of its entries'
    probabilities. The teacher gets no gradient."""
    ce, _, kd = _losses("linear_distill", h, W, y, ids, logits.detach(), float(tau))
    return kd, None if y is None else ce
