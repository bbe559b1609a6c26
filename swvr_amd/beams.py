"""Beam search's step: the best continuations over beams and vocabulary, and the states taken along.

Where ``sample_tokens`` draws one token per row, ``select_beams`` keeps the k best of all the continuations of a
sequence's beams, and ``reorder_beams`` brings the beams' states (key-value caches, token histories) into the order
of the beams that were kept:

    tokens, parents, scores = select_beams(logits, scores)       # [B, W, V], [B, W] -> [B, W] each
    reorder_beams(caches, parents, inplace=True)                 # every cache [B, W, ...]
    x = embedding_lookup(tokens, E)                              # the next step's inputs

A place for which no candidate was left has token and parent -1 and score -inf: a row of zeros in both, and no
candidates in the next step.  The kernels run on the current stream (C ABI: swvr_select_beams, swvr_reorder_beams).
"""
import ctypes
import functools
import math
from typing import List, Optional, Tuple

import torch

from . import _lib
from ._ops import _plain, _require_device, eager, no_tangents

MAX_BEAMS, MAX_IN_PLACE, MAX_V = 256, 64, 2 ** 21


# ---------------------------------------------------------------- selection
def _dense(x, dtype):
    if x is None:
        return None
    x = _plain(x)
    x = x if x.dtype == dtype else x.to(dtype)
    return x if x.is_contiguous() else x.contiguous()


@functools.lru_cache(maxsize=256)
def _workspace(B, W, V, k):
    return _lib.load().swvr_select_beams_workspace_size(B, W, V, k)


def _select(logits, scores, k, finished, end_id, lengths, alpha):
    x, (*lead, W, V) = _plain(logits), logits.shape
    x = x if x.dim() == 2 else x.reshape(-1, V)
    x = x if x.stride(1) == 1 and x.stride(0) >= 0 else x.contiguous()
    s = _dense(scores, scores.dtype if scores.dtype == torch.float64 else torch.float32)
    finished, lengths = _dense(finished, torch.bool), _dense(lengths, torch.int64)
    B, shape, ld = math.prod(lead), (*lead, k), x.stride(0) if x.shape[0] > 1 else V
    token, parent = x.new_empty(shape, dtype=torch.int64), x.new_empty(shape, dtype=torch.int64)
    out, ws_bytes = s.new_empty(shape), _workspace(B, W, V, k)
    ws, a = x.new_empty(ws_bytes, dtype=torch.uint8), _lib.address
    _lib.call(_lib.load().swvr_select_beams, x.device, _lib.DTYPE_TAG[x.dtype], B, W, V, k, x.data_ptr(), ld, s.data_ptr(),
              s.dtype == torch.float64, a(finished), end_id, a(lengths), alpha, token.data_ptr(), parent.data_ptr(),
              out.data_ptr(), ws.data_ptr(), ws_bytes)
    return token, parent, out


@torch.library.custom_op("swvr::select_beams", mutates_args=())
def _select_op(logits: torch.Tensor, scores: torch.Tensor, k: int, finished: Optional[torch.Tensor], end_id: int,
               lengths: Optional[torch.Tensor], alpha: float) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    return _select(logits, scores, k, finished, end_id, lengths, alpha)


@_select_op.register_fake
def _(logits, scores, k, finished, end_id, lengths, alpha):
    shape = (*scores.shape[:-1], k)
    kept = torch.float64 if scores.dtype == torch.float64 else torch.float32
    return (logits.new_empty(shape, dtype=torch.int64), logits.new_empty(shape, dtype=torch.int64),
            logits.new_empty(shape, dtype=kept))


def select_beams(logits, scores, k=None, *, finished=None, end_id=None, lengths=None, length_penalty=0.0):
    """The ``k`` (default W) best continuations of each sequence from ``logits`` ``[..., W, V]`` (bf16, fp16 or fp32) of
    its W beams and their ``scores`` ``[..., W]``, sums of log-probabilities: ``(tokens, parents, scores)``, each
    ``[..., k]``, best first; tokens and parents (the beam that is continued) int64, the new scores in fp32, or
    fp64 for scores in fp64.

    A candidate is a beam and a token: ``score + logit - logsumexp(logits)``.  A beam with ``finished`` (bool
    ``[..., W]``) has one, token ``end_id`` at its own score.  With ``length_penalty`` (0 to 16) candidates are
    ranked by ``score / length ** length_penalty``, the length being the beam's of ``lengths`` (integers ``[..., W]``, the
    tokens so far), with the new token unless it is finished, and at least 1; the scores given back are the sums.
    The ranks are formed in fp64, so that they order candidates of different beams as their exact values do but for
    differences of about 1e-12; equal ones come by beam, then the larger logit, then the lower token.

    NaN and -inf logits are no candidates, and a beam with a score of -inf (or one that is not finite) has none:
    scores of 0 for the first beam and -inf for the others begin a search.  A +inf logit leaves its beam without
    candidates.  Where fewer than k are left, token and parent are -1 and the score -inf.  W and k are at most 256, V
    at most 2^21.  No gradient; the same result on every run.
    """
    shape = logits.shape
    if len(shape) < 2 or not 1 <= shape[-1] <= MAX_V or not 1 <= shape[-2] <= MAX_BEAMS:
        raise ValueError(f"logits must be [..., W, V] with 1 <= W <= {MAX_BEAMS} and 1 <= V <= 2^21, got {tuple(shape)}")
    if logits.dtype not in _lib.DTYPE_TAG:
        raise NotImplementedError(f"swvr_amd: logits dtype {logits.dtype} is not supported (bf16, fp16, fp32)")
    if not scores.dtype.is_floating_point:
        raise ValueError(f"scores must be floating point, got {scores.dtype}")
    k = shape[-2] if k is None else int(k)
    if not 1 <= k <= MAX_BEAMS:
        raise ValueError(f"k must be between 1 and {MAX_BEAMS}, got {k}")
    if not 0 <= length_penalty <= 16:
        raise ValueError(f"length_penalty must be between 0 and 16, got {length_penalty}")
    if length_penalty and lengths is None:
        raise ValueError("length_penalty needs lengths")
    for name, x in (("scores", scores), ("finished", finished), ("lengths", lengths)):
        if x is None:
            continue
        if x.shape != shape[:-1]:
            raise ValueError(f"{name} must have shape {tuple(shape[:-1])}, got {tuple(x.shape)}")
        if x.device != logits.device:
            raise ValueError(f"{name} is on {x.device} but logits on {logits.device}")
    end = 0
    if finished is not None:
        if finished.dtype != torch.bool:
            raise ValueError(f"finished must be bool, got {finished.dtype}")
        if end_id is None or not 0 <= end_id < shape[-1]:
            raise ValueError(f"finished needs end_id, a token of 0 to V - 1, got {end_id}")
        end = int(end_id)
    if lengths is not None and (lengths.dtype.is_floating_point or lengths.dtype.is_complex or lengths.dtype == torch.bool):
        raise ValueError(f"lengths must be integers, got {lengths.dtype}")
    if eager(logits, scores, finished, lengths):
        return _select(logits, scores, k, finished, end, lengths, float(length_penalty))
    no_tangents(logits, scores)
    if logits.device.type == "cpu":
        _require_device(logits)
    return _select_op(logits.detach(), scores.detach(), k, finished, end, lengths, float(length_penalty))


# ---------------------------------------------------------------- states
@functools.lru_cache(maxsize=1024)
def _geometry(shape, strides, itemsize, nb):
    """Of a state [lead..., W, rest...] with nb leading dimensions: (run, n1, n2, strides, dst strides per beam of a
    dense copy's (n2, n1)), bytes; None where the kernel cannot walk them: more dimensions left after merging, or pieces
    that make 4 GB a beam."""
    def merged(dims):
        out = []
        for n, s in dims:
            if n == 1:
                continue
            if out and out[-1][1] == n * s:
                out[-1] = (out[-1][0] * n, s)
            else:
                out.append((n, s))
        return out

    dims = list(zip(shape, strides))
    lead, rest = merged(dims[:nb]), merged(dims[nb + 1:])
    run = 1
    if rest and rest[-1][1] == 1:
        run = rest.pop()[0]
    if len(lead) > 1 or len(rest) > 2 or any(s < 0 for s in strides):
        return None
    rest = [(1, 0)] * (2 - len(rest)) + rest
    (n2, s2), (n1, s1) = rest
    if n1 * n2 > 1 and run * n1 * n2 * itemsize >= 2 ** 32:   # (the library's limit of a beam in pieces)
        return None
    step = tuple(s * itemsize for s in (lead[0][1] if lead else 0, strides[nb] if shape[nb] > 1 else 0, s2, s1))
    return run * itemsize, n1, n2, step, (run * n1 * itemsize if n2 > 1 else 0, run * itemsize if n1 > 1 else 0)


@functools.lru_cache(maxsize=1024)
def _overlaps(shape, strides):
    """Whether elements of a view may share memory (as expanded ones do)."""
    reach = 0
    for s, n in sorted((s, n) for n, s in zip(shape, strides) if n > 1):
        if s <= reach:
            return True
        reach += s * (n - 1)
    return False


def _reorder(states, parents, inplace):
    ids = _plain(parents)
    ids = ids if ids.dtype in (torch.int64, torch.int32) else ids.to(torch.int64)
    ids = ids if ids.is_contiguous() else ids.contiguous()
    nb, k = ids.dim() - 1, ids.shape[-1]
    W = states[0].shape[nb]
    B = 1
    for n in ids.shape[:-1]:
        B *= n
    groups, out, kept, seen, last = {}, [], [], {parents.data_ptr()}, None
    for x in states:
        if x.is_neg() or x.is_conj() or x._is_zerotensor():
            if inplace:
                raise ValueError("a lazily negated, conjugated or memoryless state cannot be reordered in place")
            x = _plain(x.resolve_conj())
            kept.append(x)
        layout = (x.shape, x.stride(), x.element_size())
        if layout != last:   # (the caches of all layers have one)
            last, (shape, strides, _) = layout, layout
            if inplace and _overlaps(shape, strides):
                raise ValueError(f"a state with shared elements (strides {strides}) cannot be reordered in place")
            g = _geometry(*layout, nb) if x.numel() else ()
            if g is None and inplace:
                raise ValueError(f"a state of shape {tuple(shape)} with strides {strides} has too many separate dimensions (or "
                                 "pieces, of a beam of 4 GB) to be reordered in place")
            new = (*shape[:nb], k, *shape[nb + 1:])
            dense = g is None
            if dense:
                g = _geometry(shape, x.contiguous().stride(), x.element_size(), nb)
            if g:
                src, dst = groups.setdefault(g, ([], []))
        if dense:
            x = x.contiguous()
            kept.append(x)
        at = x.data_ptr()
        if inplace:
            if at in seen and g:
                raise ValueError("the same state twice, or the parents, cannot be reordered in place")
            seen.add(at)
            y = x
        else:
            y = x.new_empty(new)
            if g:
                dst.append(y.data_ptr())
        out.append(y)
        if g:
            src.append(at)
    lib = _lib.load()
    for (run, n1, n2, steps, dense), (src, dst) in groups.items():
        n = len(src)
        beam = run * n1 * n2
        at = (ctypes.c_void_p * n)(*src)
        to = None if inplace else (ctypes.c_void_p * n)(*dst)
        step = (ctypes.c_int64 * 4)(*steps)
        to_step = (ctypes.c_int64 * 4)(k * beam, beam, *dense)
        _lib.call(lib.swvr_reorder_beams, ids.device, n, at, to, B, W, k, ids.data_ptr(), ids.dtype == torch.int64, run, n1, n2,
                  step, to_step)
    return out


@torch.library.custom_op("swvr::reorder_beams", mutates_args=())
def _reorder_op(states: List[torch.Tensor], parents: torch.Tensor) -> List[torch.Tensor]:
    return _reorder(states, parents, False)


@_reorder_op.register_fake
def _(states, parents):
    nb = parents.dim() - 1
    return [torch.empty((*x.shape[:nb], parents.shape[-1], *x.shape[nb + 1:]), dtype=x.dtype, device=x.device) for x in states]


@torch.library.custom_op("swvr::reorder_beams_", mutates_args={"states"})
def _reorder_op_(states: List[torch.Tensor], parents: torch.Tensor) -> None:
    _reorder(states, parents, True)


@_reorder_op_.register_fake
def _(states, parents):
    return None


def reorder_beams(states, parents, *, inplace=False):
    """The beams' states in the order of the beams that were kept: ``out[..., j, *] = state[..., parents[..., j], *]``.

    states: a tensor, or a list or (named) tuple of them (the caches of every layer, say: those of one shape and layout are one
    launch), each ``[..., W, *]`` with the leading dimensions of ``parents`` ``[..., k]`` (integers) before the beams
    and anything after them, of any dtype; a part of a cache goes in as a view, ``cache[:, :, :, :length]``.  A parent
    outside 0 .. W - 1 (-1 of ``select_beams``, for a beam that there is none of) gives zeros.

    Gives new tensors (of the structure of ``states``), or with ``inplace`` the states themselves, reordered where they
    are: beams that keep their place are then neither read nor written.  In place k must be W, at most 64; leading
    dimensions have to be one in memory, the ones after the beams at most three after merging (one, where a beam has 4
    GB), and no element may be part of a state twice, of two states or of the parents.  No gradient: where one would be
    recorded the call is refused.
    """
    alone = isinstance(states, torch.Tensor)
    xs = [states] if alone else list(states)
    if parents.dim() < 1 or parents.dtype.is_floating_point or parents.dtype.is_complex or parents.dtype == torch.bool:
        raise ValueError(f"parents must be integers [..., k], got {parents.dtype} {tuple(parents.shape)}")
    nb, k = parents.dim() - 1, parents.shape[-1]
    if not xs:
        return states if inplace else type(states)()
    W = xs[0].shape[nb] if xs[0].dim() > nb else 0
    if not (1 <= W <= MAX_BEAMS and 1 <= k <= MAX_BEAMS):
        raise ValueError(f"states and parents must have 1 to {MAX_BEAMS} beams, got {W} and {k}")
    if inplace and (k != W or W > MAX_IN_PLACE):
        raise ValueError(f"in place as many beams come as go, at most {MAX_IN_PLACE}: got {W} and {k}")
    grad, lead, device, shape = torch.is_grad_enabled(), parents.shape[:-1], parents.device, None
    for x in xs:
        if x.shape != shape:
            shape = x.shape
            if len(shape) <= nb or shape[nb] != W or shape[:nb] != lead:
                raise ValueError(f"states must be [{', '.join(map(str, (*lead, W)))}, ...], got {tuple(shape)}")
        if x.device != device:
            raise ValueError(f"a state is on {x.device} but parents on {device}")
        if grad and x.requires_grad:
            raise ValueError("reorder_beams has no gradient: call it under torch.no_grad() or on detached tensors")
    if eager(parents, *xs):
        out = _reorder(xs, parents, inplace)
        if inplace:
            torch.autograd.graph.increment_version([x for x in xs if not x.is_inference()])
    else:
        no_tangents(*xs)
        if device.type == "cpu":
            _require_device(parents)
        if inplace:
            _reorder_op_(xs, parents)
            out = xs
        else:
            out = _reorder_op(xs, parents)
    if inplace:
        return states
    if alone:
        return out[0]
    kind = type(states)
    return kind(*out) if hasattr(kind, "_fields") else kind(out) if isinstance(states, (list, tuple)) else out
