"""The head's losses over the vocabulary, with no logits kept: cross entropy of labels and distillation from a teacher's
top logits, forward and backward on hand-written kernels (csrc/head_loss.hip; C ABI in include/lm/pragnosia_lm.h).

    loss, lse = linear_cross_entropy(h, W, y)
    kd, ce = linear_distill(h, W, ids, logits, tau, y)

h (..., d) are hidden rows and W (V, d) the head's weight (the LM's tied table), d a multiple of 8. The logits h W^T are
formed on the bf16 matrix cores in pieces of the vocabulary: h and W in another type are rounded to bf16, as autocast
rounds a Linear's operands. The reference's LM forms its logits in chunks of rows under activation checkpointing
(`src/model.py:563-567`); LM.loss does so here too, unless the model was built with fused_ends.

Every loss comes per token in fp32, so a mean, a mask or weights are the caller's own: the kernels take the per-token
gradients that autograd hands back. The gradients of logits are rounded to bf16 once, before the two products that dh
(in h's type) and dW (in W's; an fp32 W gets the unrounded fp32 sums) are; sums are held in fp32 throughout and taken in
a fixed order, so the same call gives the same bits.
"""
from __future__ import annotations

import ctypes
import math
from typing import Optional

import torch
from torch import Tensor

from ._lib import PragnosiaError, check, lm_lib
from .ops import _bf16, _expect, _f32, _ptr, _require_gpu, _stream

_FLOATS = (torch.bfloat16, torch.float32)
_INTS = (torch.int64, torch.int32, torch.int16, torch.int8, torch.uint8)


def _aligned(t: Optional[Tensor]) -> Optional[Tensor]:
    """t contiguous, at an address the kernels' 16-byte loads take (a slice of a buffer may start anywhere)."""
    if t is None:
        return None
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _check_head(op: str, h: Tensor, W: Tensor, y: Optional[Tensor], ids: Optional[Tensor], z: Optional[Tensor],
                tau: float) -> None:
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
        if ids.shape[1] == 0 or not z.is_floating_point():
            raise PragnosiaError(f"{op}: ids and logits (..., K) with K > 0 and floating logits expected, got "
                                 f"{tuple(ids.shape)} and {z.dtype}")
    if not (tau > 0 and math.isfinite(tau)):
        raise PragnosiaError(f"{op}: tau must be positive and finite, got {tau}")


@torch.library.custom_op("pragnosia::head_loss", mutates_args=())
def head_loss(h: Tensor, W: Tensor, y: Optional[Tensor], ids: Optional[Tensor], z: Optional[Tensor],
              tau: float) -> tuple[Tensor, Tensor, Tensor, Tensor, Tensor, Tensor, Tensor, Tensor, Tensor, Tensor]:
    """h (n, d), W (V, d), y (n) or None, ids and z (n, K) or None. Returns (ce, lse, kd, then what the backward takes:
    lse_t, psum, entry, p, zl, and the bf16 operands); ce and lse are empty without y, kd and its share without ids."""
    _require_gpu(h, W, y, ids, z)
    _check_head("head_loss", h, W, y, ids, z, tau)
    n, d = h.shape
    V, K = W.shape[0], 0 if ids is None else ids.shape[1]
    e = lambda *s, dt=torch.float32: torch.empty(*s, device=h.device, dtype=dt)
    ny, nk = (0 if y is None else n), (0 if ids is None else n)
    ce, lse, kd, lse_t, psum = e(ny), e(ny), e(nk), e(nk), e(nk)
    entry, p, zl = e(nk, K, dt=torch.int32), e(nk, K), e(nk, K)
    hb, Wb = h.new_empty(0), W.new_empty(0)
    if n == 0:
        return ce, lse, kd, lse_t, psum, entry, p, zl, hb, Wb
    h16, W16 = _aligned(_bf16(h)), _aligned(_bf16(W))
    y = None if y is None else y.to(torch.int64).contiguous()
    ids, z = (None, None) if ids is None else (ids.to(torch.int64).contiguous(), _f32(z))
    with torch.cuda.device(h.device):
        L = lm_lib()
        nbytes = L.pragnosia_head_fwd_workspace_bytes(n, V, d, K)
        if nbytes < 0:
            raise PragnosiaError(f"head_loss: shape n={n} V={V} d={d} K={K} rejected")
        ws = e(nbytes, dt=torch.uint8)
        opt = lambda t, on: _ptr(t) if on else None
        check(L.pragnosia_head_fwd(_ptr(h16), _ptr(W16), _ptr(y), _ptr(ids), _ptr(z), float(tau), opt(ce, ny),
                                   opt(lse, ny), opt(kd, nk), opt(lse_t, nk), opt(psum, nk), opt(entry, nk),
                                   opt(p, nk), opt(zl, nk), _ptr(ws), nbytes, n, V, d, K, _stream(h)),
              "pragnosia_head_fwd")
    return (ce, lse, kd, lse_t, psum, entry, p, zl, hb if h16.data_ptr() == h.data_ptr() else h16,
            Wb if W16.data_ptr() == W.data_ptr() else W16)


@head_loss.register_fake
def _(h, W, y, ids, z, tau):
    n, K = h.shape[0], 0 if ids is None else ids.shape[1]
    ny, nk = (0 if y is None else n), (0 if ids is None else n)
    e = lambda *s, dt=torch.float32: h.new_empty(*s, dtype=dt)
    return (e(ny), e(ny), e(nk), e(nk), e(nk), e(nk, K, dt=torch.int32), e(nk, K), e(nk, K),
            h.new_empty(0) if h.dtype == torch.bfloat16 else e(*h.shape, dt=torch.bfloat16),
            W.new_empty(0) if W.dtype == torch.bfloat16 else e(*W.shape, dt=torch.bfloat16))


@torch.library.custom_op("pragnosia::head_loss_bwd", mutates_args=())
def head_loss_bwd(g_ce: Optional[Tensor], g_lse: Optional[Tensor], g_kd: Optional[Tensor], h: Tensor, W: Tensor,
                  y: Optional[Tensor], lse: Tensor, lse_t: Tensor, psum: Tensor, entry: Tensor, p: Tensor, zl: Tensor,
                  tau: float, need_h: bool, need_W: bool, dw_f32: bool) -> tuple[Tensor, Tensor]:
    """Gradients of head_loss's ce, lse and kd -> (dh (n, d) bf16, dW (V, d) bf16 or fp32); empty where not needed. h
    and W bf16."""
    _require_gpu(g_ce, g_lse, g_kd, h, W, y, lse, lse_t, psum, entry, p, zl)
    if h.dim() != 2 or W.dim() != 2:
        raise PragnosiaError(f"head_loss_bwd: h (n, d) and W (V, d) expected, got {tuple(h.shape)}, {tuple(W.shape)}")
    n, d = h.shape
    V, K = W.shape[0], entry.shape[-1] if g_kd is not None else 0
    nk = n if g_kd is not None else None
    _expect("head_loss_bwd", h.device, W=(W, (None, d)), g_ce=(g_ce, (n,)), g_lse=(g_lse, (n,)), g_kd=(g_kd, (n,)),
            y=(y, (n,)), lse=(lse if g_ce is not None or g_lse is not None else None, (n,)))
    if g_kd is not None:
        _expect("head_loss_bwd", h.device, lse_t=(lse_t, (nk,)), psum=(psum, (nk,)), entry=(entry, (nk, K)),
                p=(p, (nk, K)), zl=(zl, (nk, K)))
    if h.dtype != torch.bfloat16 or W.dtype != torch.bfloat16 or entry.dtype != torch.int32:
        raise PragnosiaError("head_loss_bwd: h and W must be bf16 and entry int32, as head_loss returns them")
    if g_ce is not None and y is None:
        raise PragnosiaError("head_loss_bwd: g_ce without labels")
    dh = torch.empty(n if need_h else 0, d, device=h.device, dtype=torch.bfloat16)
    dW = torch.empty(V if need_W else 0, d, device=h.device, dtype=torch.float32 if dw_f32 else torch.bfloat16)
    if n == 0 or not (need_h or need_W) or (g_ce is None and g_lse is None and g_kd is None):
        return dh.zero_(), dW.zero_()
    h, W = _aligned(h), _aligned(W)
    y = None if y is None else y.to(torch.int64).contiguous()
    g_ce, g_lse, g_kd, lse, lse_t, psum, p, zl = (_f32(t) for t in (g_ce, g_lse, g_kd, lse, lse_t, psum, p, zl))
    entry = entry.contiguous()
    with torch.cuda.device(h.device):
        L = lm_lib()
        nbytes = L.pragnosia_head_bwd_workspace_bytes(n, V, d)
        if nbytes < 0:
            raise PragnosiaError(f"head_loss_bwd: shape n={n} V={V} d={d} rejected")
        ws = torch.empty(nbytes, device=h.device, dtype=torch.uint8)
        opt = lambda t, on: _ptr(t) if on else None
        kd = g_kd is not None
        check(L.pragnosia_head_bwd(_ptr(g_ce), _ptr(g_lse), _ptr(g_kd), _ptr(h), _ptr(W), _ptr(y),
                                   opt(lse, g_ce is not None or g_lse is not None), opt(lse_t, kd), opt(psum, kd),
                                   opt(entry, kd), opt(p, kd), opt(zl, kd), float(tau), opt(dh, need_h),
                                   opt(dW, need_W), int(dw_f32), _ptr(ws), nbytes, n, V, d, K, _stream(h)),
              "pragnosia_head_bwd")
    return dh, dW


@head_loss_bwd.register_fake
def _(g_ce, g_lse, g_kd, h, W, y, lse, lse_t, psum, entry, p, zl, tau, need_h, need_W, dw_f32):
    n, d = h.shape
    return (h.new_empty(n if need_h else 0, d, dtype=torch.bfloat16),
            h.new_empty(W.shape[0] if need_W else 0, d, dtype=torch.float32 if dw_f32 else torch.bfloat16))


def _head_setup(ctx, inputs, output):
    ctx.set_materialize_grads(False)  # an unused output's gradient arrives as None, not zeros
    h, W, y, ids, z, tau = inputs
    _, lse, _, lse_t, psum, entry, p, zl, h16, W16 = output
    ctx.tau, ctx.dtypes, ctx.has = tau, (h.dtype, W.dtype), (y is not None, ids is not None)
    ctx.save_for_backward(h16 if h16.dim() == 2 else h, W16 if W16.dim() == 2 else W, y, lse, lse_t, psum, entry, p, zl)
    ctx.mark_non_differentiable(lse_t, psum, entry, p, zl, h16, W16)


def _head_backward(ctx, g_ce, g_lse, g_kd, *_):
    h, W, y, lse, lse_t, psum, entry, p, zl = ctx.saved_tensors
    need_h, need_W = ctx.needs_input_grad[:2]
    has_y, has_kd = ctx.has
    dh, dW = head_loss_bwd(g_ce if has_y else None, g_lse if has_y else None, g_kd if has_kd else None, h, W, y, lse,
                           lse_t, psum, entry, p, zl, ctx.tau, need_h, need_W, ctx.dtypes[1] == torch.float32)
    return dh.to(ctx.dtypes[0]) if need_h else None, dW if need_W else None, None, None, None, None


head_loss.register_autograd(_head_backward, setup_context=_head_setup)


def _rows(op: str, h: Tensor, y: Optional[Tensor], ids: Optional[Tensor], z: Optional[Tensor]):
    lead = h.shape[:-1]
    if h.dim() < 1 or (y is not None and y.shape != lead) or any(
            t is not None and (t.dim() != h.dim() or t.shape[:-1] != lead) for t in (ids, z)):
        raise PragnosiaError(f"{op}: the labels' and the teacher's leading sizes must be h's {tuple(lead)}, got "
                             f"{[None if t is None else tuple(t.shape) for t in (y, ids, z)]}")
    flat = lambda t: None if t is None else t.reshape(-1, t.shape[-1])
    return flat(h), None if y is None else y.reshape(-1), flat(ids), flat(z)


def linear_cross_entropy(h: Tensor, W: Tensor, y: Tensor) -> tuple[Tensor, Tensor]:
    """Per-token cross entropy of the head h W^T at the labels y, and the log of the softmax's denominator (for a
    penalty on it, or a label's log-probability elsewhere): both y's shape, fp32, both differentiable in h and W.

    A label outside [0, V) (padding, such as -100) has loss 0 and adds no gradient. Such rows of h still enter dW's
    sums, times zero: they have to be finite there."""
    h2, y2, _, _ = _rows("linear_cross_entropy", h, y, None, None)
    out = head_loss(h2, W, y2, None, None, 1.0)
    return out[0].view(y.shape), out[1].view(y.shape)


def linear_distill(h: Tensor, W: Tensor, ids: Tensor, logits: Tensor, tau: float = 1.0,
                   y: Optional[Tensor] = None) -> tuple[Tensor, Optional[Tensor]]:
    """Per-token distillation loss of the head h W^T from a teacher's top logits, and with labels y the cross entropy
    (else None) from the same pass over the vocabulary; fp32, h's leading shape, differentiable in h and W.

    ids and logits (..., K): the teacher's words, in any order, and its logits there. Its distribution p is their softmax
    at temperature tau; the loss is tau^2 KL(p || q) with q the softmax of the student's logits over the whole vocabulary
    at tau. An id outside [0, V) marks an entry that is not there (lists of different lengths); a logit of -inf has
    probability zero; a token with no entry left has loss 0 and no gradient. A repeated id has the sum of its entries'
    probabilities. The teacher gets no gradient."""
    h2, y2, i2, z2 = _rows("linear_distill", h, y, ids, logits)
    out = head_loss(h2, W, y2, i2, z2.detach(), float(tau))
    return out[2].view(h.shape[:-1]), None if y is None else out[0].view(y.shape)
