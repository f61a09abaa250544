"""4-bit weights for generation, on hand-written kernels (csrc/fp4.hip; C ABI in pragnosia_amd/include/pragnosia_gen.h).

    Q = quantize(W, group)                       # W (N, K) fp32 or bf16, rounded once, before the first step
    W = dequantize(Q)                            # what it was rounded to
    y = linear(x, Q, bias, norm=ln, act="gelu", resid=r)    # gelu(ln(x) W^T + bias) + r

A weight is kept as 4-bit floating codes (e2m1: 0, 0.5, 1, 1.5, 2, 3, 4, 6 with a sign) and one bf16 scale for each group of
32, 64 or 128 columns of a row: 4.5, 4.25 or 4.125 bits a weight, decoded by the GPU's own conversion. `GreedyDecoder(model,
batch, weights="fp4")` runs a model's decode step on them; the reference decodes in fp32 (`src/bench.py:241-317`).

`linear` multiplies the values s v that the codes stand for, with fp32 sums, and is as exact as its operands' type lets it
be: fp32 rows, and normalised rows of either type, are not rounded (they go through the bf16 matrix cores in three parts),
other bf16 rows are taken as they are. Values of a row may lie between 2^-102, below which their last bits may be lost, and
2^118, past which a group's sum may overflow before its scale. Sums are taken in a fixed order: the same call gives the same
bits.

There is no backward: `linear` refuses an input that requires a gradient where gradients are recorded. `quantize` takes the
present values of a weight, also of a parameter that is being trained; no gradient leads back through the codes. An eager
call goes straight to the C ABI; one that something records or replaces (torch.compile, make_fx, torch.export,
torch.jit.trace, a dispatch mode) goes through the custom ops `pragnosia_gen::fp4_*`.
"""
from __future__ import annotations

from typing import Optional

import torch
from torch import Tensor
from torch.autograd import forward_ad

from ._lib import PragnosiaError, check, gen_lib
from .head import _BF16, _F32, _FLOATS, _as, _at, _call, _no_tangents, _raw_stream, _watched
from .ops import _expect, _require_gpu

GROUPS = (32, 64, 128)
_ACTS = {None: 0, "gelu": 1}
_U8, _empty = torch.uint8, torch.empty
_device = torch._C._cuda_getDevice  # current_device() without the check that CUDA is initialised: a GPU tensor was made


class Weight4:
    """A weight (N, K) in 4 bits: `codes` (uint8) and `scales` (bf16) as the kernels lay them out, `group` columns to a
    scale, and `dtype`, the type it was rounded from."""

    __slots__ = ("codes", "scales", "N", "K", "group", "dtype")

    def __init__(self, codes: Tensor, scales: Tensor, N: int, K: int, group: int, dtype: torch.dtype = _F32):
        _check_weight("Weight4", codes, scales, N, K, group)
        self._set(codes, scales, N, K, group, dtype)

    def _set(self, codes, scales, N, K, group, dtype):
        # (written out: torch.compile traces these and `Weight4.__new__(Weight4)`, and no other names for them)
        object.__setattr__(self, "codes", codes), object.__setattr__(self, "scales", scales)
        object.__setattr__(self, "dtype", dtype), object.__setattr__(self, "N", N)
        object.__setattr__(self, "K", K), object.__setattr__(self, "group", group)
        return self

    def __setattr__(self, name, value):
        raise PragnosiaError(f"Weight4: {name} cannot be changed (its sizes were checked together)")

    def __reduce__(self):  # copies and pickles go through the checks too
        return Weight4, (self.codes, self.scales, self.N, self.K, self.group, self.dtype)

    @property
    def shape(self):
        return torch.Size((self.N, self.K))

    @property
    def device(self):
        return self.codes.device

    @property
    def nbytes(self) -> int:
        return self.codes.numel() + 2 * self.scales.numel()

    def __repr__(self):
        return f"Weight4({self.N}, {self.K}, group={self.group}, {self.device})"


def _sizes(op: str, N: int, K: int, group: int) -> tuple[int, int]:
    """Bytes of codes and number of scales of a weight (N, K); refuses what the kernels do not take."""
    if group not in GROUPS:
        raise PragnosiaError(f"{op}: group must be one of {GROUPS}, got {group}")
    if not (0 < N <= 1 << 26 and 0 < K <= 65536 and K % 8 == 0):
        raise PragnosiaError(f"{op}: a weight (N, K) with N from 1 to 2^26 and K a multiple of 8 up to 65536 expected, "
                             f"got ({N}, {K})")
    tiles = -(-N // 16) * -(-K // 128)
    return tiles * 1024, tiles * 16 * (128 // group)


def _check_weight(op: str, codes: Tensor, scales: Tensor, N: int, K: int, group: int) -> None:
    nbytes, count = _sizes(op, N, K, group)
    for name, t, dt, size in (("codes", codes, torch.uint8, nbytes), ("scales", scales, _BF16, count)):
        if t.dtype != dt or tuple(t.shape) != (size,) or not t.is_contiguous() or t.data_ptr() % 16:
            raise PragnosiaError(f"{op}: {name} of ({N}, {K}) at group {group} must be {size} dense {dt}, 16-byte aligned, "
                                 f"got {tuple(t.shape)} {t.dtype}")
    if codes.device != scales.device:
        raise PragnosiaError(f"{op}: codes on {codes.device}, scales on {scales.device}")


def _quantize(W: Tensor, group: int, codes: Tensor, scales: Tensor) -> None:
    W = _as(W.detach(), W.dtype)
    _call("pragnosia_fp4_quantize", gen_lib().pragnosia_fp4_quantize, W, _at(W), W.dtype == _BF16, _at(codes),
          _at(scales), W.shape[0], W.shape[1], group)


def _dequantize(codes: Tensor, scales: Tensor, N: int, K: int, group: int, dtype: torch.dtype) -> Tensor:
    W = torch.empty(N, K, device=codes.device, dtype=dtype)
    _call("pragnosia_fp4_dequantize", gen_lib().pragnosia_fp4_dequantize, W, _at(codes), _at(scales), _at(W),
          dtype == _BF16, N, K, group)
    return W


def _check_source(op: str, W: Tensor, group: int) -> tuple[int, int]:
    _require_gpu(W)
    if W.dim() != 2 or W.dtype not in _FLOATS:
        raise PragnosiaError(f"{op}: a weight (N, K) in fp32 or bf16 expected, got {tuple(W.shape)} {W.dtype}")
    _no_tangents(op, W)
    return _sizes(op, W.shape[0], W.shape[1], group)


def quantize(W: Tensor, group: int = 64, out: Optional[Weight4] = None) -> Weight4:
    """W (N, K), fp32 or bf16, in 4 bits with a scale for each `group` (32, 64 or 128) columns of a row. A scale is
    max |w| / 6 rounded to bf16, a code the nearest value (ties to the even code, past 6 to 6); a group with an infinity or
    a NaN becomes NaN throughout. A W that requires a gradient is detached. `out`: a Weight4 of the same sizes, group and
    device to write into (one that a captured graph reads, say)."""
    # the usual call, without the general path's looks at everything (10 us of host; this 7)
    if W.dim() == 2 and out is None and _quiet({type(W)}):
        index, dt, (N, K) = W.get_device(), W.dtype, W.shape
        if (W.is_cuda and index == _device() and dt in _FLOATS and group in GROUPS and 0 < N <= 1 << 26 and 0 < K <= 65536
                and K % 8 == 0 and W.is_contiguous() and not W.data_ptr() & 15 and forward_ad._current_level < 0):
            tiles = -(-N // 16) * -(-K // 128)
            codes = _empty(tiles * 1024, device=W.device, dtype=_U8)
            scales = _empty(tiles * (2048 // group), device=W.device, dtype=_BF16)
            rc = gen_lib().pragnosia_fp4_quantize(W.data_ptr(), dt is _BF16, codes.data_ptr(), scales.data_ptr(), N, K, group,
                                                  _raw_stream(index))
            if rc:
                check(rc, "pragnosia_fp4_quantize")
            return Weight4.__new__(Weight4)._set(codes, scales, N, K, group, dt)
    nbytes, count = _check_source("quantize", W, group)
    N, K = W.shape
    if out is not None:
        if tuple(out.shape) != (N, K) or out.group != group or out.device != W.device:
            raise PragnosiaError(f"quantize: out is {out}, expected ({N}, {K}) at group {group} on {W.device}")
        if _watched(W):
            raise PragnosiaError("quantize: `out` is not available in a trace or under a dispatch mode")
        _quantize(W, group, out.codes, out.scales)
        return out._set(out.codes, out.scales, N, K, group, W.dtype)
    if _watched(W):
        codes, scales = fp4_quantize(W.detach(), group)
    else:
        codes = torch.empty(nbytes, device=W.device, dtype=torch.uint8)
        scales = torch.empty(count, device=W.device, dtype=_BF16)
        _quantize(W, group, codes, scales)
    return Weight4.__new__(Weight4)._set(codes, scales, N, K, group, W.dtype)  # (sizes are right by construction)


def dequantize(Q: Weight4, dtype: Optional[torch.dtype] = None) -> Tensor:
    """The weight that Q stands for, (N, K): exactly in fp32, rounded once in bf16 (the type it came from by default)."""
    dtype = dtype or Q.dtype
    if dtype not in _FLOATS:
        raise PragnosiaError(f"dequantize: fp32 or bf16 expected, got {dtype}")
    codes, scales = Q.codes, Q.scales
    index = codes.get_device()
    if _quiet({type(codes), type(scales)}) and codes.is_cuda and index == _device():
        W = _empty(Q.N, Q.K, device=codes.device, dtype=dtype)
        rc = gen_lib().pragnosia_fp4_dequantize(codes.data_ptr(), scales.data_ptr(), W.data_ptr(), dtype is _BF16, Q.N, Q.K,
                                                Q.group, _raw_stream(index))
        if rc:
            check(rc, "pragnosia_fp4_dequantize")
        return W
    _require_gpu(Q.codes)
    if _watched(Q.codes, Q.scales):
        return fp4_dequantize(Q.codes, Q.scales, Q.N, Q.K, Q.group, dtype == _BF16)
    return _dequantize(Q.codes, Q.scales, Q.N, Q.K, Q.group, dtype)


def _fits(t: Tensor, dt: torch.dtype, index: int, shape: tuple) -> bool:
    """Whether the kernels take t, on GPU `index`, as it is."""
    return (t.dtype is dt and t.get_device() == index and t.shape == shape and t.is_contiguous()
            and not t.data_ptr() & 15)


_PLAIN = {Tensor, torch.nn.Parameter, type(None), float, int}


def _quiet(types: set) -> bool:
    """_watched's negative, of a set of argument types. Asked before anything else of a short way: what stands behind it (the
    current device, addresses) is neither traced nor there for a fake tensor."""
    return not _watched() and _PLAIN.issuperset(types)


def _linear(x: Tensor, codes: Tensor, scales: Tensor, lnw: Optional[Tensor], lnb: Optional[Tensor], eps: float,
            bias: Optional[Tensor], act: int, resid: Optional[Tensor], N: int, group: int) -> Tensor:
    """x (n, K) and the rest checked, all of x's type."""
    n, K = x.shape
    dt = x.dtype
    x, lnw, lnb, bias, resid = _as(x, dt), _as(lnw, dt), _as(lnb, dt), _as(bias, dt), _as(resid, dt)
    y = torch.empty(n, N, device=x.device, dtype=dt)
    if n:
        _call("pragnosia_fp4_linear", gen_lib().pragnosia_fp4_linear, x, _at(x), dt is _BF16, _at(codes), _at(scales),
              _at(lnw), _at(lnb), eps, _at(bias), act, _at(resid), _at(y), n, N, K, group)
    return y


def _check_linear(op: str, x: Tensor, codes: Tensor, scales: Tensor, lnw: Optional[Tensor], lnb: Optional[Tensor],
                  eps: float, bias: Optional[Tensor], resid: Optional[Tensor], N: int, K: int) -> None:
    _require_gpu(x, codes, scales, lnw, lnb, bias, resid)
    if x.dtype not in _FLOATS:
        raise PragnosiaError(f"{op}: x must be fp32 or bf16, got {x.dtype}")
    n = x.shape[0] if x.dim() == 2 else None
    _expect(op, x.device, x=(x, (None, K)), codes=(codes, (None,)), scales=(scales, (None,)), ln_weight=(lnw, (K,)),
            ln_bias=(lnb, (K,)), bias=(bias, (N,)), resid=(resid, (n, N)))
    for name, t in (("ln_weight", lnw), ("ln_bias", lnb), ("bias", bias), ("resid", resid)):
        if t is not None and t.dtype not in _FLOATS:
            raise PragnosiaError(f"{op}: {name} must be fp32 or bf16, got {t.dtype}")
    if lnw is None and lnb is not None:
        raise PragnosiaError(f"{op}: a LayerNorm without a weight has no bias here")
    if not eps >= 0.0:
        raise PragnosiaError(f"{op}: the norm's eps must not be negative, got {eps}")
    if n > 1 << 24 or n * max(N, K) >= 1 << 31:
        raise PragnosiaError(f"{op}: at most 2^24 rows, and fewer than 2^31 values in and out, got {n} rows of {K} and {N}")


def linear(x: Tensor, Q: Weight4, bias: Optional[Tensor] = None, *, norm: Optional[torch.nn.LayerNorm] = None,
           act: Optional[str] = None, resid: Optional[Tensor] = None) -> Tensor:
    """act(norm(x) W^T + bias) + resid with the weight that Q stands for: x (..., K) fp32 or bf16, result (..., N) in its
    type. norm: an affine LayerNorm over K; act: None or "gelu" (erf form); bias (N) and resid (..., N). Parameters and resid
    of the other type are rounded to x's. For inference: any input that requires a gradient is refused where gradients are
    recorded."""
    N, K = Q.N, Q.K
    lnw, lnb, eps = None, None, 0.0
    if norm is not None:
        if not isinstance(norm, torch.nn.LayerNorm) or tuple(norm.normalized_shape) != (K,) or norm.weight is None:
            raise PragnosiaError(f"linear: norm must be an affine LayerNorm over {K}, got {norm}")
        lnw, lnb, eps = norm.weight, norm.bias, norm.eps
    if act not in _ACTS:
        raise PragnosiaError(f"linear: act must be None or 'gelu', got {act!r}")
    if x.dim() == 0 or x.shape[-1] == 0 or (resid is not None and resid.shape != (*x.shape[:-1], N)):
        raise PragnosiaError(f"linear: x (..., {K}) and resid (..., {N}) expected, got {tuple(x.shape)} and "
                             f"{None if resid is None else tuple(resid.shape)}")
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, lnw, lnb, bias, resid)):
        raise PragnosiaError("linear: 4-bit weights have no backward; call it under torch.no_grad()")
    _no_tangents("linear", x, lnw, lnb, bias, resid)
    # the usual call: nothing to convert, to refuse or to record, and the host has no more to do than to see so (the general
    # path below takes 15 us of the host for a projection of one row, this one 9, its launch 5 of either)
    dt, index, n = x.dtype, x.get_device(), x.shape[0]
    if (_quiet({type(x), type(lnw), type(lnb), type(bias), type(resid), type(Q.codes), type(Q.scales)})
            and x.is_cuda and x.dim() == 2 and 0 < n <= 1 << 16 and n * max(N, K) < 1 << 31 and dt in _FLOATS and eps >= 0.0
            and index == Q.codes.get_device() == _device() and _fits(x, dt, index, (n, K))
            and (lnw is None or _fits(lnw, dt, index, (K,)) and (lnb is None or _fits(lnb, dt, index, (K,))))
            and (bias is None or _fits(bias, dt, index, (N,))) and (resid is None or _fits(resid, dt, index, (n, N)))):
        y = x.new_empty(n, N)
        rc = gen_lib().pragnosia_fp4_linear(x.data_ptr(), dt is _BF16, Q.codes.data_ptr(), Q.scales.data_ptr(), _at(lnw),
                                            _at(lnb), eps, _at(bias), _ACTS[act], _at(resid), y.data_ptr(), n, N, K,
                                            Q.group, _raw_stream(index))
        if rc:
            check(rc, "pragnosia_fp4_linear")
        return y
    flat = x if x.dim() == 2 else x.reshape(-1, x.shape[-1])
    r = resid if resid is None or resid.dim() == 2 else resid.reshape(-1, N)
    _check_linear("linear", flat, Q.codes, Q.scales, lnw, lnb, eps, bias, r, N, K)
    if _watched(flat, Q.codes, Q.scales, lnw, lnb, bias, r):
        y = fp4_linear(flat, Q.codes, Q.scales, lnw, lnb, eps, bias, _ACTS[act], r, N, Q.group)
    else:
        y = _linear(flat, Q.codes, Q.scales, lnw, lnb, eps, bias, _ACTS[act], r, N, Q.group)
    return y if x.dim() == 2 else y.view(*x.shape[:-1], N)


# ---------------------------------------------------------------------------------------------------------------
# the same as custom ops, for traces
@torch.library.custom_op("pragnosia_gen::fp4_quantize", mutates_args=())
def fp4_quantize(W: Tensor, group: int) -> tuple[Tensor, Tensor]:
    """W (N, K) -> (codes uint8, scales bf16), laid out for the kernels."""
    nbytes, count = _check_source("fp4_quantize", W, group)
    codes = torch.empty(nbytes, device=W.device, dtype=torch.uint8)
    scales = torch.empty(count, device=W.device, dtype=_BF16)
    _quantize(W, group, codes, scales)
    return codes, scales


@fp4_quantize.register_fake
def _(W, group):
    tiles = -(-W.shape[0] // 16) * -(-W.shape[1] // 128)
    return W.new_empty(tiles * 1024, dtype=torch.uint8), W.new_empty(tiles * 16 * (128 // group), dtype=_BF16)


@torch.library.custom_op("pragnosia_gen::fp4_dequantize", mutates_args=())
def fp4_dequantize(codes: Tensor, scales: Tensor, N: int, K: int, group: int, bf16: bool) -> Tensor:
    """(codes, scales) of a weight (N, K) -> the weight, fp32 or bf16."""
    _require_gpu(codes, scales)
    _check_weight("fp4_dequantize", codes, scales, N, K, group)
    return _dequantize(codes, scales, N, K, group, _BF16 if bf16 else _F32)


@fp4_dequantize.register_fake
def _(codes, scales, N, K, group, bf16):
    return codes.new_empty(N, K, dtype=_BF16 if bf16 else _F32)


@torch.library.custom_op("pragnosia_gen::fp4_linear", mutates_args=())
def fp4_linear(x: Tensor, codes: Tensor, scales: Tensor, lnw: Optional[Tensor], lnb: Optional[Tensor], eps: float,
               bias: Optional[Tensor], act: int, resid: Optional[Tensor], N: int, group: int) -> Tensor:
    """x (n, K) times a weight (N, K) in 4 bits, with the norm, bias, activation (0: none, 1: GELU) and residual."""
    if x.dim() != 2 or act not in (0, 1):
        raise PragnosiaError(f"fp4_linear: x (n, K) and act 0 or 1 expected, got {tuple(x.shape)} and {act}")
    _check_weight("fp4_linear", codes, scales, N, x.shape[1], group)
    _check_linear("fp4_linear", x, codes, scales, lnw, lnb, eps, bias, resid, N, x.shape[1])
    _no_tangents("fp4_linear", x, lnw, lnb, bias, resid)
    return _linear(x, codes, scales, lnw, lnb, float(eps), bias, act, resid, N, group)


@fp4_linear.register_fake
def _(x, codes, scales, lnw, lnb, eps, bias, act, resid, N, group):
    return x.new_empty(x.shape[0], N)
