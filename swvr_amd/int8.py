"""The head in 8-bit integers, for serving: logits at a byte per weight.

``sample_tokens`` and ``select_beams`` take logits.  ``head_logits`` makes them from a head whose rows are held as
integers with a scale each, ``W[v] ~ scale[v] * q[v]``; h is quantised the same way, a scale per token, within the
call, and the sum over K is exact in 32-bit integers.

    w = int8.quantize_rows(W)                     # once; or int8.pack_rows(q, scale) for integers quantised elsewhere
    logits = int8.head_logits(h, w, bias)         # every step

Beside the e4m3 readout (``swvr_amd.fp8``) this is opt-in and outside the reference's precision policy
(swvr/chunked.py:7-9): exact for the integers, while rounding h and W to 127 steps of their rows' largest values adds
its own error to the logits.  The kernels run on the current stream (C ABI: swvr_int8_quantize, swvr_int8_pack,
swvr_int8_unpack, swvr_int8_logits).
"""
from typing import NamedTuple, Optional, Tuple

import torch

from . import _lib
from ._ops import _plain, _require_device, eager, no_tangents

K_MAX, ROWS_MAX = 2 ** 17, 2 ** 25


class Int8Rows(NamedTuple):
    """Rows held in integers: ``q`` in the layout of the matrix cores (the library's own, int8), ``scale`` [R] in fp32,
    and the rows' ``shape`` (R, K)."""
    q: torch.Tensor
    scale: torch.Tensor
    shape: Tuple[int, int]


def _image_shape(R, K):
    return (R + 255) // 256 * 8, (K + 63) // 64, 2048


def _rows(x):
    """``x`` [R, K] with unit inner stride and rows in order."""
    x = _plain(x)
    return x if x.stride(1) == 1 and x.stride(0) >= 0 else x.contiguous()


def _ld(x):
    return x.stride(0) if x.shape[0] > 1 else x.shape[1]


def _quantize(x):
    x = _rows(x)
    R, K = x.shape
    q = x.new_empty(_image_shape(R, K), dtype=torch.int8)
    scale = x.new_empty(R, dtype=torch.float32)
    _lib.call(_lib.load().swvr_int8_quantize, x.device, _lib.DTYPE_TAG[x.dtype], R, K, x.data_ptr(), _ld(x), q.data_ptr(),
              scale.data_ptr())
    return q, scale


def _pack(x, scale):
    x = _rows(x)
    R, K = x.shape
    q, kept = x.new_empty(_image_shape(R, K)), x.new_empty(R, dtype=torch.float32)
    kept.copy_(scale)
    _lib.call(_lib.load().swvr_int8_pack, x.device, R, K, x.data_ptr(), _ld(x), q.data_ptr())
    return q, kept


def _unpack(q, scale, R, K):
    out = scale.new_empty(R, K)
    _lib.call(_lib.load().swvr_int8_unpack, q.device, R, K, q.data_ptr(), scale.data_ptr(), out.data_ptr())
    return out


def _logits(h, q, scale, bias, V, logit_scale, dtype):
    x = _rows(h if h.dim() == 2 else h.reshape(-1, h.shape[-1]))
    N, K = x.shape
    lib = _lib.load()
    out = x.new_empty(*h.shape[:-1], V, dtype=dtype)
    b_tag = 0
    if bias is not None:
        bias = _plain(bias)
        bias = bias if bias.dtype in _lib.DTYPE_TAG else bias.to(torch.float32)
        bias = bias if bias.is_contiguous() else bias.contiguous()
        b_tag = _lib.DTYPE_TAG[bias.dtype]
    ws_bytes = lib.swvr_int8_logits_workspace_size(N, K)
    ws = x.new_empty(ws_bytes, dtype=torch.uint8)
    _lib.call(lib.swvr_int8_logits, x.device, _lib.DTYPE_TAG[x.dtype], _lib.DTYPE_TAG[dtype], N, K, V, x.data_ptr(), _ld(x),
              q.data_ptr(), scale.data_ptr(), _lib.address(bias), b_tag, logit_scale, out.data_ptr(), ws.data_ptr(), ws_bytes)
    return out


@torch.library.custom_op("swvr::int8_quantize", mutates_args=())
def _quantize_op(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    return _quantize(x)


@_quantize_op.register_fake
def _(x):
    return x.new_empty(_image_shape(*x.shape), dtype=torch.int8), x.new_empty(x.shape[0], dtype=torch.float32)


@torch.library.custom_op("swvr::int8_pack", mutates_args=())
def _pack_op(x: torch.Tensor, scale: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    return _pack(x, scale)


@_pack_op.register_fake
def _(x, scale):
    return x.new_empty(_image_shape(*x.shape)), x.new_empty(x.shape[0], dtype=torch.float32)


@torch.library.custom_op("swvr::int8_unpack", mutates_args=())
def _unpack_op(q: torch.Tensor, scale: torch.Tensor, R: int, K: int) -> torch.Tensor:
    return _unpack(q, scale, R, K)


@_unpack_op.register_fake
def _(q, scale, R, K):
    return scale.new_empty(R, K)


@torch.library.custom_op("swvr::int8_logits", mutates_args=())
def _logits_op(h: torch.Tensor, q: torch.Tensor, scale: torch.Tensor, bias: Optional[torch.Tensor], V: int,
               logit_scale: float, dtype: torch.dtype) -> torch.Tensor:
    return _logits(h, q, scale, bias, V, logit_scale, dtype)


@_logits_op.register_fake
def _(h, q, scale, bias, V, logit_scale, dtype):
    return h.new_empty(*h.shape[:-1], V, dtype=dtype)


def _sizes(name, x):
    if x.dim() != 2:
        raise ValueError(f"{name} must be 2-D, got {tuple(x.shape)}")
    if not 1 <= x.shape[1] <= K_MAX or x.shape[0] > ROWS_MAX:
        raise ValueError(f"{name} must have 1 to 2^17 columns and at most 2^25 rows, got {tuple(x.shape)}")


def _no_gradient(what, *tensors):
    no_tangents(*tensors)
    if torch.is_grad_enabled():
        for t in tensors:  # (a loop, as in eager)
            if t is not None and t.requires_grad:
                raise ValueError(f"{what} has no gradient: call it under torch.no_grad() or on detached tensors")


def quantize_rows(x):
    """``Int8Rows`` of a matrix ``x`` [R, K] in bf16, fp16 or fp32: ``scale = max(amax, 1e-30) * fl(1/127)`` per row in
    fp32 and ``q = x / scale`` rounded to the nearest whole number (halves to even, by the exact quotient).  A row with
    an infinity or a NaN gets scale NaN.  No gradient: ``x`` is detached, as a parameter is when it is quantised once."""
    _sizes("x", x)
    if x.dtype not in _lib.DTYPE_TAG:
        raise NotImplementedError(f"swvr_amd: rows of {x.dtype} are not supported (bf16, fp16, fp32)")
    no_tangents(x)
    x = x.detach()
    if eager(x):
        q, scale = _quantize(x)
    else:
        if x.device.type == "cpu":
            _require_device(x)
        q, scale = _quantize_op(x)
    return Int8Rows(q, scale, (x.shape[0], x.shape[1]))


def pack_rows(q, scale):
    """``Int8Rows`` from integers ``q`` [R, K] (int8, as a file holds them) and their scales [R]; both are copied."""
    _sizes("q", q)
    if q.dtype != torch.int8:
        raise ValueError(f"q must be int8, got {q.dtype}")
    if scale.shape != q.shape[:1] or not scale.dtype.is_floating_point:
        raise ValueError(f"scale must be floating point of shape {tuple(q.shape[:1])}, got {scale.dtype} {tuple(scale.shape)}")
    if scale.device != q.device:
        raise ValueError(f"scale is on {scale.device} but q on {q.device}")
    no_tangents(scale)
    scale = scale.detach()
    if eager(q, scale):
        q8, kept = _pack(q, scale)
    else:
        if q.device.type == "cpu":
            _require_device(q)
        q8, kept = _pack_op(q, scale)
    return Int8Rows(q8, kept, (q.shape[0], q.shape[1]))


def _checked(w):
    """(q, scale, R, K) of an ``Int8Rows`` that fits together."""
    if not isinstance(w, Int8Rows):
        raise ValueError(f"w must be what quantize_rows or pack_rows gave, got {type(w).__name__}")
    q, scale, (R, K) = w
    if q.dtype != torch.int8 or tuple(q.shape) != _image_shape(R, K) or scale.dtype != torch.float32 or \
            tuple(scale.shape) != (R,) or scale.device != q.device:
        raise ValueError(f"w does not fit together: q {q.dtype} {tuple(q.shape)}, scale {scale.dtype} {tuple(scale.shape)} "
                         f"for {R} rows of {K}")
    if not (q.is_contiguous() and scale.is_contiguous()):
        raise ValueError("w must be as quantize_rows or pack_rows gave it, got strided views")
    return q, scale, R, K


def dequantize(w):
    """The values that ``w`` stands for, ``scale * q``, in fp32 [R, K].  No gradient: where the scales would record one the
    call is refused."""
    q, scale, R, K = _checked(w)
    _no_gradient("dequantize", scale)
    if eager(q, scale):
        return _unpack(q, scale, R, K)
    if q.device.type == "cpu":
        _require_device(q)
    return _unpack_op(q, scale, R, K)


def head_logits(h, w, bias=None, *, logit_scale=1.0, dtype=None):
    """Logits ``logit_scale * h @ W.T + bias`` of a head held in integers: ``[..., V]`` in ``dtype`` (bf16, fp16 or
    fp32; None: h's own).

    h: ``[..., K]`` in bf16, fp16 or fp32 (up to 2^24 tokens), quantised per token as ``quantize_rows`` does; w:
    ``quantize_rows(W)`` or ``pack_rows(q, scale)`` of the [V, K] head; bias: ``[V]``.  The sum over K is exact, the
    scales and the bias are applied in fp32 (in fp64 where the product of the scales leaves its range), and the result
    is rounded once.  A token's logits do not depend on the
    others in the call.  A token or a row of W with an infinity or a NaN has NaN logits.  There is no gradient: where one
    would be recorded the call is refused.
    """
    q, scale, V, K = _checked(w)
    if h.dim() < 1 or h.shape[-1] != K:
        raise ValueError(f"h must be [..., {K}], got {tuple(h.shape)}")
    if h.dtype not in _lib.DTYPE_TAG:
        raise NotImplementedError(f"swvr_amd: h of {h.dtype} is not supported (bf16, fp16, fp32)")
    dtype = h.dtype if dtype is None else dtype
    if dtype not in _lib.DTYPE_TAG:
        raise NotImplementedError(f"swvr_amd: logits of {dtype} are not supported (bf16, fp16, fp32)")
    if bias is not None and (bias.shape != (V,) or not bias.dtype.is_floating_point):
        raise ValueError(f"bias must be floating point of shape ({V},), got {bias.dtype} {tuple(bias.shape)}")
    for name, x in (("w", q), ("bias", bias)):
        if x is not None and x.device != h.device:
            raise ValueError(f"{name} is on {x.device} but h on {h.device}")
    _no_gradient("head_logits", h, scale, bias)
    if eager(h, q, scale, bias):
        return _logits(h, q, scale, bias, V, float(logit_scale), dtype)
    if h.device.type == "cpu":
        _require_device(h)
    return _logits_op(h, q, scale, bias, V, float(logit_scale), dtype)
