"""Lookup of token rows with a scale, and its gradient by sorted tokens, on hand-written kernels (csrc/embed.hip; C ABI
in pragnosia_amd/include/pragnosia_lm.h).

    y = embedding(ids, W, scale)

is scale * W[ids] with a zero row where an id is outside the table (padding). The gradient of W is summed in fp32 over a
stable order of the tokens by id: no atomics on values, so the same bits each time, and no memset in a captured step,
where torch's embedding sorts with one from some thousands of indices on (`src/model.py:822-826` is the reference's
lookup)."""
from __future__ import annotations

import math
from typing import Optional

import torch
from torch import Tensor

from ._lib import PragnosiaError, lm_lib
from .head import (_BF16, _F32, _FLOATS, _I64, _INTS, _as, _at, _call, _no_tangents, _once, _watched,
                   _workspace)
from .ops import _expect, _require_gpu


def _check_embed(op: str, ids: Tensor, W: Tensor, scale: float, dtype: torch.dtype) -> None:
    _require_gpu(ids, W)
    if ids.dtype not in _INTS:
        raise PragnosiaError(f"{op}: ids must be integers, got {ids.dtype}")
    _expect(op, W.device, ids=(ids, (None,)), W=(W, (None, None)))
    if W.dtype not in _FLOATS or dtype not in _FLOATS:
        raise PragnosiaError(f"{op}: the table and the rows must be bf16 or fp32, got {W.dtype} and {dtype}")
    if W.shape[0] == 0 or W.shape[1] == 0 or W.shape[1] % 8:
        raise PragnosiaError(f"{op}: a table (V, d) with V > 0 and d a multiple of 8 expected, got {tuple(W.shape)}")
    if not math.isfinite(scale):
        raise PragnosiaError(f"{op}: scale must be finite, got {scale}")


def _forward(ids: Tensor, W: Tensor, scale: float, dtype: torch.dtype, kept: Optional[Tensor] = None) -> Tensor:
    """ids (n) int64, W (V, d), both contiguous. kept: (n) int32 for the ids as the backward takes them, or None."""
    n, (V, d) = ids.shape[0], W.shape
    y = torch.empty(n, d, device=W.device, dtype=dtype)
    _call("pragnosia_embed_fwd", lm_lib().pragnosia_embed_fwd, W, _at(ids), _at(W), W.dtype == _BF16, scale, _at(y),
          dtype == _BF16, _at(kept), n, V, d)
    return y


def _backward(g: Tensor, ids: Tensor, V: int, scale: float, dtype: torch.dtype) -> Tensor:
    """g (n, d), ids (n) int64 or int32 -> dW (V, d) in `dtype`."""
    g = _as(g, g.dtype)
    n, d = g.shape
    dW = torch.empty(V, d, device=g.device, dtype=dtype)
    nbytes = _workspace("pragnosia_embed_bwd_workspace_bytes", n, V, d)
    ws = torch.empty(nbytes, device=g.device, dtype=torch.uint8) if nbytes else None
    _call("pragnosia_embed_bwd", lm_lib().pragnosia_embed_bwd, g, _at(g), g.dtype == _BF16, _at(ids), ids.dtype == _I64,
          scale, _at(dW), dtype == _BF16, _at(ws), nbytes, n, V, d)
    return dW


# Tokens from which the lookup keeps the ids in 32 bits: every sorting workgroup reads them all. Lookup and gradient,
# 768 wide, without and with: 65536 tokens of 512 words 182 and 155 us, of 32768 words 328 and 323; 32768 of 32768 182
# and 179; up to 16384 within 1.3 us, which the host's allocation of them takes. (A traced call keeps none.)
_KEPT_FROM = 16385


class _Embedding(torch.autograd.Function):
    @staticmethod
    def forward(ctx, ids, W, scale, dtype):
        ids, n = _as(ids, _I64), ids.shape[0]
        kept = torch.empty(n, device=W.device, dtype=torch.int32) if n >= _KEPT_FROM else None
        ctx.save_for_backward(ids if kept is None else kept)
        ctx.V, ctx.scale, ctx.dtype = W.shape[0], scale, W.dtype
        return _forward(ids, _as(W, W.dtype), scale, dtype, kept)

    @staticmethod
    @_once
    def backward(ctx, g):
        _no_tangents("embed_bwd", g)
        ids, = ctx.saved_tensors
        if _watched(g):
            return None, embed_bwd(g, ids, ctx.V, ctx.scale, ctx.dtype == _BF16), None, None
        return None, _backward(g, ids, ctx.V, ctx.scale, ctx.dtype), None, None


# ---------------------------------------------------------------------------------------------------------------
# the same as custom ops, for traces
@torch.library.custom_op("pragnosia_lm::embed", mutates_args=())
def embed(ids: Tensor, W: Tensor, scale: float, bf16: bool) -> Tensor:
    """ids (n), W (V, d) -> scale W[ids] (n, d), bf16 or fp32."""
    dtype = _BF16 if bf16 else _F32
    _check_embed("embed", ids, W, scale, dtype)
    _no_tangents("embed", W)
    return _forward(_as(ids, _I64), _as(W, W.dtype), float(scale), dtype)


@embed.register_fake
def _(ids, W, scale, bf16):
    return W.new_empty(ids.shape[0], W.shape[1], dtype=_BF16 if bf16 else _F32)


@torch.library.custom_op("pragnosia_lm::embed_bwd", mutates_args=())
def embed_bwd(g: Tensor, ids: Tensor, V: int, scale: float, bf16: bool) -> Tensor:
    """g (n, d), ids (n) -> dW (V, d), bf16 or fp32."""
    _require_gpu(g, ids)
    _no_tangents("embed_bwd", g)
    if g.dtype not in _FLOATS or g.dim() != 2 or g.shape[1] % 8 or g.shape[1] == 0 or V <= 0:
        raise PragnosiaError(f"embed_bwd: gradients (n, d) in bf16 or fp32 expected, got {tuple(g.shape)} {g.dtype}")
    if ids.dtype not in _INTS:
        raise PragnosiaError(f"embed_bwd: ids must be integers, got {ids.dtype}")
    _expect("embed_bwd", g.device, ids=(ids, (g.shape[0],)))
    return _backward(g, _as(ids, _I64), V, float(scale), _BF16 if bf16 else _F32)


@embed_bwd.register_fake
def _(g, ids, V, scale, bf16):
    return g.new_empty(V, g.shape[1], dtype=_BF16 if bf16 else _F32)


def _embed_setup(ctx, inputs, output):
    ids, W, scale, _ = inputs
    ctx.save_for_backward(ids)
    ctx.V, ctx.scale, ctx.bf16 = W.shape[0], scale, W.dtype == _BF16


def _embed_backward(ctx, g):
    ids, = ctx.saved_tensors
    return None, embed_bwd(g, ids, ctx.V, ctx.scale, ctx.bf16), None, None


embed.register_autograd(_embed_backward, setup_context=_embed_setup)


def embedding(ids: Tensor, W: Tensor, scale: float = 1.0, dtype: Optional[torch.dtype] = None) -> Tensor:
    """scale * W[ids], (..., d) in `dtype` (W's by default; the product is rounded once). W (V, d) bf16 or fp32, d a
    multiple of 8. An id outside [0, V) gives a row of zeros and takes no part in W's gradient."""
    dtype, scale = dtype or W.dtype, float(scale)
    _no_tangents("embedding", W)
    flat = ids if ids.dim() == 1 else ids.reshape(-1)
    # (the usual call, without the checks' share of a short one)
    if not (W.is_cuda and flat.device == W.device and flat.dtype is _I64 and W.dim() == 2 and W.dtype in _FLOATS
            and dtype in _FLOATS and W.shape[0] > 0 and W.shape[1] > 0 and W.shape[1] % 8 == 0
            and math.isfinite(scale)):
        _check_embed("embedding", flat, W, scale, dtype)
    if _watched(flat, W):
        y = embed(flat, W, scale, dtype == _BF16)
    elif torch.is_grad_enabled() and W.requires_grad:
        y = _Embedding.apply(flat, W, scale, dtype)
    else:
        y = _forward(_as(flat, _I64), _as(W, W.dtype), scale, dtype)
    return y if ids.dim() == 1 else y.view(*ids.shape, W.shape[-1])
