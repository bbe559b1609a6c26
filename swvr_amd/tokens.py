"""Tokens in place of distributions: the lookup of a token's embedding and the draw of a token from logits.

``softmax_readout`` mixes the embedding rows of a whole distribution.  A model that is also trained or
run on tokens needs the two ends of that by themselves: ``embedding_lookup`` is the readout of a one-hot
distribution (with the table's gradient summed in a fixed order, like every gradient here), and
``sample_tokens`` picks the token.  A token of -1, which ``sample_tokens`` gives for a row with nothing
to draw, is padding for ``embedding_lookup``: a row of zeros.

The kernels run on the current stream (C ABI: swvr_embedding, swvr_embedding_bwd, swvr_sample).
"""
import math
from typing import Optional, Tuple

import torch

from . import _lib
from ._ops import _plain, _require_device, eager, first_order, no_tangents

_EMBED_TAG = {**_lib.DTYPE_TAG, torch.float64: _lib.F64}
_SORT_FREE = 2048  # tokens up to which the gradient needs neither order nor workspace (their sizes are 0)


# ---------------------------------------------------------------- embedding lookup
def _ids(ids):
    """``ids`` as a dense int32 or int64 vector."""
    if ids.dtype != torch.int64 and ids.dtype != torch.int32:
        ids = ids.to(torch.int64)
    ids = ids if ids.dim() == 1 else ids.reshape(-1)
    return ids if ids.is_contiguous() else ids.contiguous()


def _lookup(ids, E, scale, sort=False):
    """The rows, and with ``sort`` (for the gradient) the tokens' order that ``_lookup_grad`` takes, else None (few
    tokens need none)."""
    lib = _lib.load()
    i, x = _ids(ids), _plain(E)
    V, D = x.shape
    if not x.is_contiguous() and (x.stride(1) != 1 or (V > 1 and x.stride(0) < D)):
        x = x.contiguous()
    N = i.numel()
    out = x.new_empty(*ids.shape, D)
    order = None
    if sort and N > _SORT_FREE:
        order = x.new_empty(lib.swvr_embedding_sorted_size(N, V), dtype=torch.uint8)
    _lib.call(lib.swvr_embedding, x.device, _EMBED_TAG[x.dtype], i.dtype == torch.int64, N, V, D, i.data_ptr(),
              x.data_ptr(), x.stride(0) if V > 1 else D, scale, out.data_ptr(), _lib.address(order))
    return out, order


def _lookup_grad(g, ids, V, scale, order=None):
    lib = _lib.load()
    D = g.shape[-1]
    i, g2 = _ids(ids), _plain(g)
    g2 = g2 if g2.dim() == 2 else g2.reshape(i.numel(), D)
    g2 = g2 if g2.stride(1) == 1 else g2.contiguous()
    tag, N = _EMBED_TAG[g.dtype], i.numel()
    gE = g2.new_empty(V, D)
    ws, ws_bytes = None, 0
    if N > _SORT_FREE:
        ws_bytes = lib.swvr_embedding_bwd_workspace_size(tag, N, V, D)
        ws = g2.new_empty(ws_bytes, dtype=torch.uint8)
    a = _lib.address
    _lib.call(lib.swvr_embedding_bwd, g2.device, tag, i.dtype == torch.int64, N, V, D, i.data_ptr(), g2.data_ptr(),
              g2.stride(0), scale, a(order), gE.data_ptr(), a(ws), ws_bytes)
    return gE


@torch.library.custom_op("swvr::embedding", mutates_args=())
def _lookup_op(ids: torch.Tensor, E: torch.Tensor, scale: float) -> torch.Tensor:
    return _lookup(ids, E, scale)[0]


@_lookup_op.register_fake
def _(ids, E, scale):
    return E.new_empty(*ids.shape, E.shape[1])


@torch.library.custom_op("swvr::embedding_bwd", mutates_args=())
def _lookup_grad_op(g: torch.Tensor, ids: torch.Tensor, V: int, scale: float) -> torch.Tensor:
    return _lookup_grad(g, ids, V, scale)


@_lookup_grad_op.register_fake
def _(g, ids, V, scale):
    return g.new_empty(V, g.shape[-1])


def _lookup_setup(ctx, inputs, output):
    ids, E, scale = inputs
    ctx.save_for_backward(ids)
    ctx.args = (E.shape[0], scale)


def _lookup_autograd(ctx, g):
    (ids,) = ctx.saved_tensors
    return None, _lookup_grad_op(g, ids, *ctx.args) if ctx.needs_input_grad[1] else None, None


_lookup_op.register_autograd(_lookup_autograd, setup_context=_lookup_setup)


class _Lookup(torch.autograd.Function):
    """swvr::embedding / embedding_bwd as one node; the ids are sorted with the forward, whose launches cost the
    host less than those from autograd's thread."""

    @staticmethod
    def forward(ctx, ids, E, scale):
        out, order = _lookup(ids, E, scale, True)
        ctx.save_for_backward(ids, order)
        ctx.args = (E.shape[0], scale)
        return out

    @staticmethod
    @first_order
    def backward(ctx, g):
        ids, order = ctx.saved_tensors
        if eager(g, ids):
            return None, _lookup_grad(g, ids, *ctx.args, order), None
        return None, _lookup_grad_op(g, ids, *ctx.args), None


def embedding_lookup(ids, E, *, scale=1.0):
    """Rows of the embedding table: ``scale * E[ids]``, shape ``ids.shape + (D,)``, in E's dtype.

    ids: integers of any shape; E: ``[V, D]`` (each up to 2^30) in bf16, fp16, fp32 or fp64.  The product is
    formed in fp32, with scale in fp32 (fp64 for fp64), and rounded to E's dtype.  A negative id is padding: a row
    of zeros, and no share in the gradient.  Nothing can be raised for an id of V or more without waiting for the
    GPU: its row is NaN, and no row of the gradient is its.  E's gradient is dense, each row the sum of its
    tokens' cotangents in fp32 (fp64 for fp64), in an order that depends on the ids alone, so it is the same on
    every run.
    """
    if E.dim() != 2:
        raise ValueError(f"E must be 2-D, got {tuple(E.shape)}")
    if ids.dtype.is_floating_point or ids.dtype.is_complex or ids.dtype == torch.bool:
        raise ValueError(f"ids must be integers, got {ids.dtype}")
    if E.dtype not in _EMBED_TAG:
        raise NotImplementedError(f"swvr_amd: embedding dtype {E.dtype} is not supported (bf16, fp16, fp32, fp64)")
    if ids.device != E.device:
        raise ValueError(f"ids are on {ids.device} but E on {E.device}")
    if eager(ids, E):
        if E.requires_grad and torch.is_grad_enabled():
            return _Lookup.apply(ids, E, float(scale))
        return _lookup(ids, E, scale)[0]
    no_tangents(E)
    if E.device.type == "cpu":
        _require_device(E)
    return _lookup_op(ids, E, float(scale))


# ---------------------------------------------------------------- sampling
def _per_row(x, dtype, R):
    """A setting of a row each as a dense vector, or None for one value for all."""
    if x is None:
        return None
    x = _plain(x).reshape(R)
    if x.dtype != dtype:
        # (top_k: any k of 0 or less is all, and so is one past V, which is below 2^31)
        x = (x.to(torch.int64).clamp(0, 2 ** 31 - 1) if dtype == torch.int32 else x).to(dtype)
    return x if x.is_contiguous() else x.contiguous()


def _sample(logits, u, tau, k, p, min_p, tau_r, k_r, p_r, min_p_r):
    x, R, V = _plain(logits), u.numel(), logits.shape[-1]
    x = x if x.dim() == 2 else x.reshape(R, V)
    x = x if x.stride(1) == 1 else x.contiguous()
    u1 = _per_row(u, u.dtype if u.dtype == torch.float64 else torch.float32, R)
    tau_r, k_r = _per_row(tau_r, torch.float32, R), _per_row(k_r, torch.int32, R)
    p_r, min_p_r = _per_row(p_r, torch.float32, R), _per_row(min_p_r, torch.float32, R)
    token, logprob = x.new_empty(u.shape, dtype=torch.int64), x.new_empty(u.shape, dtype=torch.float32)
    a, lib = _lib.address, _lib.load()
    ws_bytes = lib.swvr_sample_workspace_size(R, V)
    ws = x.new_empty(ws_bytes, dtype=torch.uint8)
    _lib.call(lib.swvr_sample, x.device, _lib.DTYPE_TAG[x.dtype], R, V, x.data_ptr(), x.stride(0),
              u1.data_ptr(), u1.dtype == torch.float64, tau, a(tau_r), k, a(k_r), p, a(p_r), min_p, a(min_p_r),
              token.data_ptr(), logprob.data_ptr(), ws.data_ptr(), ws_bytes)
    return token, logprob


@torch.library.custom_op("swvr::sample", mutates_args=())
def _sample_op(logits: torch.Tensor, u: torch.Tensor, tau: float, k: int, p: float, min_p: float,
               tau_r: Optional[torch.Tensor], k_r: Optional[torch.Tensor], p_r: Optional[torch.Tensor],
               min_p_r: Optional[torch.Tensor]) -> Tuple[torch.Tensor, torch.Tensor]:
    return _sample(logits, u, tau, k, p, min_p, tau_r, k_r, p_r, min_p_r)


@_sample_op.register_fake
def _(logits, u, tau, k, p, min_p, tau_r, k_r, p_r, min_p_r):
    return u.new_empty(u.shape, dtype=torch.int64), u.new_empty(u.shape, dtype=torch.float32)


def _setting(name, x, default, lo, hi, u):
    """(value for all rows, tensor of one per row or None), checked."""
    if isinstance(x, torch.Tensor):
        if x.shape != u.shape:
            raise ValueError(f"{name} must be a number or have u's shape {tuple(u.shape)}, got {tuple(x.shape)}")
        if x.device != u.device:
            raise ValueError(f"{name} is on {x.device} but u on {u.device}")
        if name == "top_k" and (x.dtype.is_floating_point or x.dtype == torch.bool):
            raise ValueError(f"top_k must be integers, got {x.dtype}")
        return default, x
    if x is None:
        return default, None
    if not lo <= x <= hi:
        raise ValueError(f"{name} must be between {lo} and {hi}, got {x}")
    return type(default)(min(x, 2 ** 62)), None


def sample_tokens(logits, u, *, temperature=1.0, top_k=None, top_p=None, min_p=None):
    """One token per row of ``logits`` ``[..., V]`` (bf16, fp16 or fp32) from uniform numbers ``u`` ``[...]`` in
    [0, 1): ``(tokens, logprobs)``, int64 and fp32 of u's shape.

    A row's tokens are ordered by logit (larger first, equal ones by index); with weights
    ``w = exp((logit - largest) / temperature)``, ``top_k`` keeps the first k of them (0 or None: all), ``top_p``
    of those the ones before which the sum of w is below ``top_p`` times their sum (1 or None: all), and
    ``min_p`` those with ``w >= min_p``; the first is always kept.  The token drawn is the first by index whose
    running sum of kept weights exceeds ``u`` times their sum; its logprob is under the kept distribution.
    A temperature of 0 takes the first token (logprob 0).  -inf and NaN logits are never drawn; a row
    of nothing else gives token -1 and logprob -inf.

    Each setting is a number, or a tensor of u's shape with one per row (temperature, top_p and min_p are read
    as fp32; a temperature below 0 or NaN counts as 0, a min_p above 1 as 1).  The same u, logits and settings give
    the same token on every run and in any batch: the sums are exact.  No gradient.
    """
    if logits.dim() < 1 or logits.shape[-1] < 1:
        raise ValueError(f"logits must be [..., V] with V >= 1, got {tuple(logits.shape)}")
    if u.shape != logits.shape[:-1]:
        raise ValueError(f"u must have shape {tuple(logits.shape[:-1])}, got {tuple(u.shape)}")
    if not u.dtype.is_floating_point:
        raise ValueError(f"u must be floating point, got {u.dtype}")
    if logits.dtype not in _lib.DTYPE_TAG:
        raise NotImplementedError(f"swvr_amd: logits dtype {logits.dtype} is not supported (bf16, fp16, fp32)")
    if u.device != logits.device:
        raise ValueError(f"u is on {u.device} but logits on {logits.device}")
    tau, tau_r = _setting("temperature", temperature, 1.0, 0, 3e38, u)
    k, k_r = _setting("top_k", top_k, 0, 0, math.inf, u)
    p, p_r = _setting("top_p", top_p, 1.0, 0, 1, u)
    mp, mp_r = _setting("min_p", min_p, 0.0, 0, 1, u)
    if eager(logits, u, tau_r, k_r, p_r, mp_r):
        return _sample(logits.detach(), u, tau, k, p, mp, tau_r, k_r, p_r, mp_r)
    if logits.device.type == "cpu":
        _require_device(logits)
    return _sample_op(logits.detach(), u.detach(), tau, k, p, mp, tau_r, k_r, p_r, mp_r)
