"""Distillation of the head from a teacher's top logits, without a [tokens, V] matrix for many tokens.

Where ``softmax_readout_mse`` trains the readout O against target vectors, ``softmax_distill`` trains the
distribution itself against the part of a teacher's that is kept: its largest logits and their ids, the way
teacher outputs are stored.  One entry per token is cross entropy.  The log-normaliser and the dense part of
the gradients run on the readout's kernels (no embedding), the teacher's entries on their own (C ABI:
swvr_distill, swvr_distill_bwd).
"""
from typing import List, Optional, Tuple

import torch

from . import _lib
from ._ops import (DEFAULT_CHUNK, REDUCTIONS, _f32, _grad_buffer, _kpad, _lead_stride, _needs_grad, _operand, _plain,
                   _require_device, _rows_staged, eager, first_order, no_tangents)
from .api import _chunk, _compute_dtype

MAX_TEACHER = 1024


def _lists(x, keep, other):
    """Teacher logits or ids as [N, T] with unit inner stride, in one of the dtypes ``keep`` or as ``other``."""
    x = _plain(x)
    x = x if x.dtype in keep else x.to(other)
    return x if x.stride(1) == 1 and x.stride(0) >= 0 else x.contiguous()


def _kept(kept, N, T, need_grad):
    """Addresses in the fp32 buffer a call keeps: c [1], lse [N], and for the gradient coef [N], p [N, T], q [N, T]."""
    at = kept.data_ptr()
    lse, coef = at + 4, at + 4 * (1 + N)
    return (at, lse, coef, coef + 4 * N, coef + 4 * (N + N * T)) if need_grad else (at, lse, None, None, None)


def _forward(h, W, bias, teacher, ids, weight, tau, z, reduction, scale, chunk, cdt, need_grad, alias=True):
    """The loss, what ``_kept`` names, the bias over tau in fp32 (empty without a bias; with ``alias``, at tau = 1
    an fp32 bias itself), and the scores where the library keeps them for the backward (few tokens, no chunk
    given; else empty)."""
    lib = _lib.load()
    N, K = h.shape
    V, T = W.shape[0], ids.shape[1]
    Kp = _kpad(K)
    (hc, h_tag), (Wc, w_tag) = _operand(h, cdt, Kp), _operand(W, cdt, Kp)
    b, w = _bias(bias), _f32(weight)
    t = _lists(teacher, _lib.DTYPE_TAG, torch.float32)
    i = _lists(ids, (torch.int64, torch.int32), torch.int64)
    tag = _lib.DTYPE_TAG[cdt]
    out = hc.new_empty((N,) if reduction == 0 else (), dtype=torch.float32)
    kept = hc.new_empty(1 + N * (2 * T + 2) if need_grad else 1 + N, dtype=torch.float32)
    if alias and b is not None and tau == 1 and b.dtype == torch.float32:
        sb = b
    else:
        sb = hc.new_empty(V if b is not None else 0, dtype=torch.float32)
    scores = None
    if need_grad and chunk is None:
        kept_bytes = lib.swvr_distill_scores_size(tag, w_tag, N, Kp, V, _lead_stride(Wc))
        # a forward that keeps them computes the tokens of weight zero too: not where that costs most (half of 3000
        # dropped, K = 256, V = 30000: 1079 us without, 1168 with them)
        if w is not None and kept_bytes > 2 * V * Kp * Wc.element_size():
            kept_bytes = 0
        scores = hc.new_empty(kept_bytes // 4, dtype=torch.float32) if kept_bytes else None
    ws_bytes = lib.swvr_distill_workspace_size(tag, N, Kp, V, T, w is not None and scores is None)
    ws = hc.new_empty(ws_bytes, dtype=torch.uint8)
    a = _lib.address
    c, lse, coef, p, q = _kept(kept, N, T, need_grad)
    _lib.call(lib.swvr_distill, h.device, tag, h_tag, w_tag, N, Kp, V, T, hc.data_ptr(), _lead_stride(hc),
              Wc.data_ptr(), _lead_stride(Wc), a(b), _lib.DTYPE_TAG[b.dtype] if b is not None else 0, sb.data_ptr(),
              scale, i.data_ptr(), i.dtype == torch.int64, i.stride(0), t.data_ptr(), _lib.DTYPE_TAG[t.dtype],
              t.stride(0), tau, a(w), z, reduction, out.data_ptr(), c, lse, p, q, coef, a(scores), ws.data_ptr(),
              ws_bytes)
    return out, kept, sb, scores


def _bias(bias):
    """``bias`` dense, in a dtype the library reads (or None)."""
    if bias is None:
        return None
    b = _plain(bias)
    return (b if b.dtype in _lib.DTYPE_TAG else b.to(torch.float32)).contiguous()


def _backward(g, h, W, bias, ids, kept, sb, scores, tau, z, reduction, scale, chunk, cdt, need_h, need_W, need_b):
    lib = _lib.load()
    N, K = h.shape
    V, T = W.shape[0], ids.shape[1]
    Kp = _kpad(K)
    (hc, h_tag), (Wc, w_tag) = _operand(h, cdt, Kp), _operand(W, cdt, Kp)
    g32 = _f32(g)
    i = _lists(ids, (torch.int64, torch.int32), torch.int64)
    dev = h.device
    gh = _grad_buffer((N, Kp), h.dtype, dev) if need_h else None
    gW = _grad_buffer((V, Kp), W.dtype, dev) if need_W else None
    gb = _grad_buffer((V,), bias.dtype, dev) if need_b else None
    tag = _lib.DTYPE_TAG[cdt]
    chunk = _rows_staged(chunk, tag, w_tag, N, Kp, V, 0, need_h)
    ws_bytes = lib.swvr_distill_bwd_workspace_size(tag, w_tag, N, Kp, V, T, chunk, need_h)
    ws = hc.new_empty(ws_bytes, dtype=torch.uint8)

    def of(x):
        return (x.data_ptr(), _lib.DTYPE_TAG[x.dtype]) if x is not None else (None, 0)

    c, lse, coef, p, q = _kept(kept, N, T, True)
    _lib.call(lib.swvr_distill_bwd, dev, tag, h_tag, w_tag, N, Kp, V, T, hc.data_ptr(), _lead_stride(hc),
              Wc.data_ptr(), _lead_stride(Wc), sb.data_ptr() if bias is not None else None, scale, i.data_ptr(),
              i.dtype == torch.int64, i.stride(0), tau, z, reduction, g32.data_ptr(), c, lse, p, q, coef,
              _lib.address(scores), chunk, *of(gh), *of(gW), *of(gb), ws.data_ptr(), ws_bytes)
    if gh is not None:
        gh = gh[:, :K] if Kp != K else gh
        gh = gh.to(h.dtype) if gh.dtype != h.dtype else gh
    if gW is not None:
        gW = gW[:, :K].contiguous() if Kp != K else gW
        gW = gW.to(W.dtype) if gW.dtype != W.dtype else gW
    if gb is not None and gb.dtype != bias.dtype:
        gb = gb.to(bias.dtype)
    return gh, gW, gb


@torch.library.custom_op("swvr::distill", mutates_args=())
def _fwd_op(h: torch.Tensor, W: torch.Tensor, bias: Optional[torch.Tensor], teacher: torch.Tensor, ids: torch.Tensor,
            weight: Optional[torch.Tensor], tau: float, z: float, reduction: int, scale: float, chunk: int,
            cdt: torch.dtype, need_grad: bool) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    return _forward(h, W, bias, teacher, ids, weight, tau, z, reduction, scale, chunk, cdt, need_grad,
                    alias=False)[:3]


@_fwd_op.register_fake
def _(h, W, bias, teacher, ids, weight, tau, z, reduction, scale, chunk, cdt, need_grad):
    N, T = ids.shape

    def new(*shape):
        return h.new_empty(shape, dtype=torch.float32)

    return (new(N) if reduction == 0 else new(), new(1 + N * (2 * T + 2) if need_grad else 1 + N),
            new(W.shape[0] if bias is not None else 0))


@torch.library.custom_op("swvr::distill_bwd", mutates_args=())
def _bwd_op(g: torch.Tensor, h: torch.Tensor, W: torch.Tensor, bias: Optional[torch.Tensor], ids: torch.Tensor,
            kept: torch.Tensor, sb: torch.Tensor, tau: float, z: float, reduction: int, scale: float, chunk: int,
            cdt: torch.dtype, need_h: bool, need_W: bool, need_b: bool) -> List[torch.Tensor]:
    grads = _backward(g, h, W, bias, ids, kept, sb, None, tau, z, reduction, scale, chunk, cdt, need_h, need_W, need_b)
    # a custom op cannot return None: an empty tensor stands for "no gradient" (and dense ones, as traced: h's with
    # padded rows is a view)
    return [x.contiguous() if x is not None else h.new_empty(0) for x in grads]


@_bwd_op.register_fake
def _(g, h, W, bias, ids, kept, sb, tau, z, reduction, scale, chunk, cdt, need_h, need_W, need_b):
    # (dense whatever the parameter's layout)
    return [torch.empty(x.shape, dtype=x.dtype, device=x.device) if need else h.new_empty(0)
            for need, x in ((need_h, h), (need_W, W), (need_b, bias))]


def _setup_context(ctx, inputs, output):
    h, W, bias, _, ids, _, tau, z, reduction, scale, chunk, cdt, _ = inputs
    _, kept, sb = output
    ctx.mark_non_differentiable(kept, sb)
    ctx.save_for_backward(h, W, bias, ids, kept, sb)
    ctx.args = (tau, z, reduction, scale, chunk, cdt)


def _needs(ctx, bias):
    need_h, need_W, need_b = ctx.needs_input_grad[:3]
    return need_h, need_W, need_b and bias is not None


def _op_grads(g, saved, args, needs):
    *args, chunk, cdt = args
    grads = _bwd_op(g, *saved, *args, chunk or DEFAULT_CHUNK, cdt, *needs)
    return [x if need else None for x, need in zip(grads, needs)]


def _autograd_backward(ctx, g, *_):
    saved = ctx.saved_tensors
    return (*_op_grads(g, saved, ctx.args, _needs(ctx, saved[2])), *[None] * 10)


_fwd_op.register_autograd(_autograd_backward, setup_context=_setup_context)


class _Distill(torch.autograd.Function):
    """swvr::distill / distill_bwd as one node, returning the loss."""

    @staticmethod
    def forward(ctx, h, W, bias, teacher, ids, weight, tau, z, reduction, scale, chunk, cdt):
        out, kept, sb, scores = _forward(h, W, bias, teacher, ids, weight, tau, z, reduction, scale, chunk, cdt, True)
        ctx.save_for_backward(h, W, bias, ids, kept, sb, scores)
        ctx.args = (tau, z, reduction, scale, chunk, cdt)
        return out

    @staticmethod
    @first_order
    def backward(ctx, g):
        saved = ctx.saved_tensors
        needs = _needs(ctx, saved[2])
        if eager(g, *saved):
            grads = _backward(g, *saved, *ctx.args, *needs)
        else:
            grads = _op_grads(g, saved[:-1], ctx.args, needs)
        return (*grads, *[None] * 9)


def _check(h, W, teacher, ids, bias, weight, temperature, reduction):
    if W.dim() != 2 or W.shape[0] < 1:
        raise ValueError(f"W must be 2-D with at least one row, got {tuple(W.shape)}")
    if h.dim() < 1 or h.shape[-1] != W.shape[1]:
        raise ValueError(f"h has shape {tuple(h.shape)} but W is {tuple(W.shape)}")
    if bias is not None and bias.shape != (W.shape[0],):
        raise ValueError(f"bias must have shape ({W.shape[0]},), got {tuple(bias.shape)}")
    lead = h.shape[:-1]
    if ids.shape != teacher.shape or ids.dim() < 1 or ids.shape[:-1] != lead:
        raise ValueError(f"teacher_logits and teacher_ids must both be {tuple(lead)} + (T,), got "
                         f"{tuple(teacher.shape)} and {tuple(ids.shape)}")
    if not 1 <= ids.shape[-1] <= MAX_TEACHER:
        raise ValueError(f"a teacher's list holds 1 to {MAX_TEACHER} entries, got {ids.shape[-1]}")
    if ids.dtype.is_floating_point or ids.dtype.is_complex or ids.dtype == torch.bool:
        raise ValueError(f"teacher_ids must be integers, got {ids.dtype}")
    if not teacher.dtype.is_floating_point:
        raise ValueError(f"teacher_logits must be floating point, got {teacher.dtype}")
    if weight is not None and weight.shape != lead:
        raise ValueError(f"weight must have shape {tuple(lead)}, got {tuple(weight.shape)}")
    for name, x in (("W", W), ("teacher_logits", teacher), ("teacher_ids", ids), ("bias", bias), ("weight", weight)):
        if x is not None and x.device != h.device:
            raise ValueError(f"{name} is on {x.device} but h on {h.device}")
    for name, x in (("teacher_logits", teacher), ("weight", weight)):
        if x is not None and x.requires_grad:
            raise ValueError(f"{name} gets no gradient: detach it")
    if not 4e-39 < temperature < 3e38:  # (its reciprocal is held in fp32 too)
        raise ValueError(f"temperature must be between 4e-39 and 3e38, got {temperature}")
    if reduction not in REDUCTIONS:
        raise ValueError(f"unknown reduction {reduction!r}")


def softmax_distill(h, W, teacher_logits, teacher_ids, bias=None, *, temperature=1.0, weight=None, reduction="mean",
                    z_loss_weight=0.0, logit_scale=1.0, chunk_size=None):
    """Divergence of the head's distribution from a teacher's top logits.

    With student scores ``S = (logit_scale * h W^T + bias) / temperature`` over the V vocabulary rows (h ``[..., K]``,
    W ``[V, K]``, optional bias ``[V]``), ``LSE = logsumexp(S)``, and the teacher's distribution
    ``p = softmax(teacher_logits / temperature)`` over the T (1 to 1024) entries it gives for a token
    (``teacher_logits`` and integer ``teacher_ids``, both ``[..., T]``), each token contributes
    ``sum_k p_k (log p_k - S[id_k] + LSE)``, plus ``z_loss_weight * LSE^2``.  One entry per token is cross entropy.
    An entry with a negative id or a logit of -inf is absent; ids may repeat.  A token without entries
    contributes nothing.  An id of V or more makes its token's term NaN, and with it the gradients that the token
    reaches: its row of h's, all of W's and bias's.

    ``weight`` (``[...]``) multiplies each term; a zero drops the token, whatever its inputs hold.  ``reduction``:
    "mean" (the weighted sum over the sum of the weights of the tokens that have an entry; 0 without any),
    "sum" or "none" (the per-token terms).  The loss is fp32; there is no factor of ``temperature ** 2``.  The
    products run in autocast's dtype or the promotion of h's and W's (bf16, fp16 or fp32), and the backward
    recomputes the scores ``chunk_size`` vocabulary rows at a time, as ``softmax_readout`` does.  An eager call
    without a chunk, and with W in the products' dtype (fp32 parameters under autocast are not), keeps the scores of
    few tokens (up to 768, in fp32 any number) for it instead, where they take at most 512 MB and twice W's bytes (K
    tokens in the 2-byte types, 2 K in fp32; in fp32 without a weight, any number of tokens from K = 128 on).
    Autograd reaches h, W and bias; the teacher and the weight get none.  In fp16 the gradients, and the softmax's
    part of them, fall below the type's range where many tokens share a mean: scale the loss, as fp16 training does.
    """
    _check(h, W, teacher_logits, teacher_ids, bias, weight, temperature, reduction)
    chunk = _chunk(chunk_size)
    cdt = _compute_dtype(h, W)
    if cdt not in _lib.DTYPE_TAG:
        raise NotImplementedError(f"swvr_amd: compute dtype {cdt} is not supported here (bf16, fp16, fp32)")
    lead, T = h.shape[:-1], teacher_ids.shape[-1]
    h2 = h.reshape(-1, h.shape[-1]) if h.dim() != 2 else h
    t2, i2 = teacher_logits.reshape(-1, T), teacher_ids.reshape(-1, T)
    w1 = weight.reshape(-1) if weight is not None else None
    red = REDUCTIONS[reduction]
    args = (float(temperature), float(z_loss_weight), red, float(logit_scale))
    need = _needs_grad(h, W, bias)
    if eager(h, W, teacher_logits, teacher_ids, bias, weight):
        if need:
            out = _Distill.apply(h2, W, bias, t2, i2, w1, *args, chunk, cdt)
        else:
            out = _forward(h2, W, bias, t2, i2, w1, *args, chunk, cdt, False)[0]
    else:
        no_tangents(h, W, teacher_logits, bias, weight)
        if h.device.type == "cpu":
            _require_device(h)
        if h.device.type == "cuda":
            with torch.autocast(h.device.type, enabled=False):
                out = _fwd_op(h2, W, bias, t2, i2, w1, *args, chunk or DEFAULT_CHUNK, cdt, need)[0]
        else:  # meta / fake tracing: no autocast state
            out = _fwd_op(h2, W, bias, t2, i2, w1, *args, chunk or DEFAULT_CHUNK, cdt, need)[0]
    return out.view(lead) if red == 0 else out
