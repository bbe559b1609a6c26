"""Host-side checks of the decoding operators that need no GPU: refused arguments, shapes under tracing, and the C ABI's
own checks (nothing is launched)."""
import collections
import ctypes

import pytest
import torch

import swvr_amd
from swvr_amd import _lib, int8
from swvr_amd.beams import _geometry, _overlaps

X, S = torch.zeros(2, 3, 9), torch.zeros(2, 3)
F, N = torch.zeros(2, 3, dtype=torch.bool), torch.zeros(2, 3, dtype=torch.int64)
P, C = torch.zeros(2, 3, dtype=torch.int64), torch.zeros(2, 3, 4, 5)
META = dict(device="meta")


def rows(R=9, K=16, device="cpu", **kw):
    q, s = torch.zeros(int8._image_shape(R, K), dtype=torch.int8, device=device), torch.zeros(R, device=device)
    return int8.Int8Rows(kw.get("q", q), kw.get("scale", s), kw.get("shape", (R, K)))


H = torch.zeros(4, 16)


@pytest.mark.parametrize("call", [
    lambda: swvr_amd.select_beams(torch.zeros(9), torch.zeros(())),
    lambda: swvr_amd.select_beams(torch.zeros(2, 3, 0), S),
    lambda: swvr_amd.select_beams(torch.zeros(2, 0, 9), torch.zeros(2, 0)),
    lambda: swvr_amd.select_beams(torch.zeros(1, 257, 2), torch.zeros(1, 257)),
    lambda: swvr_amd.select_beams(torch.zeros(1, 1, 2 ** 21 + 1, **META), torch.zeros(1, 1, **META)),
    lambda: swvr_amd.select_beams(X, S[:, :2]),
    lambda: swvr_amd.select_beams(X, N),
    lambda: swvr_amd.select_beams(X, S, 0),
    lambda: swvr_amd.select_beams(X, S, -1),
    lambda: swvr_amd.select_beams(X, S, 257),
    lambda: swvr_amd.select_beams(X, S, finished=F),
    lambda: swvr_amd.select_beams(X, S, finished=F, end_id=9),
    lambda: swvr_amd.select_beams(X, S, finished=F, end_id=-1),
    lambda: swvr_amd.select_beams(X, S, finished=N, end_id=1),
    lambda: swvr_amd.select_beams(X, S, finished=F[:1], end_id=1),
    lambda: swvr_amd.select_beams(X, S, lengths=N[:1]),
    lambda: swvr_amd.select_beams(X, S, lengths=S),
    lambda: swvr_amd.select_beams(X, S, lengths=F),
    lambda: swvr_amd.select_beams(X, S, length_penalty=0.5),
    lambda: swvr_amd.select_beams(X, S, lengths=N, length_penalty=-0.1),
    lambda: swvr_amd.select_beams(X, S, lengths=N, length_penalty=16.5),
    lambda: swvr_amd.select_beams(X, S, lengths=N, length_penalty=float("nan")),
    lambda: swvr_amd.select_beams(X, torch.zeros(2, 3, **META)),
    lambda: swvr_amd.select_beams(X, S, lengths=torch.zeros(2, 3, dtype=torch.int64, **META)),
    lambda: swvr_amd.reorder_beams(C, S),
    lambda: swvr_amd.reorder_beams(C, F),
    lambda: swvr_amd.reorder_beams(C, torch.zeros((), dtype=torch.int64)),
    lambda: swvr_amd.reorder_beams(C, P[:1]),
    lambda: swvr_amd.reorder_beams(C, torch.zeros(2, 0, dtype=torch.int64)),
    lambda: swvr_amd.reorder_beams(C, torch.zeros(2, 257, dtype=torch.int64)),
    lambda: swvr_amd.reorder_beams(torch.zeros(2, 0, 4), P),
    lambda: swvr_amd.reorder_beams(torch.zeros(2), P),
    lambda: swvr_amd.reorder_beams([C, torch.zeros(2, 4, 5)], P),
    lambda: swvr_amd.reorder_beams(C, torch.zeros(2, 4, dtype=torch.int64), inplace=True),
    lambda: swvr_amd.reorder_beams(torch.zeros(2, 65, 4), torch.zeros(2, 65, dtype=torch.int64), inplace=True),
    lambda: swvr_amd.reorder_beams([C, C.to("meta")], P),
    lambda: swvr_amd.reorder_beams(C.clone().requires_grad_(True), P),
    lambda: int8.quantize_rows(torch.zeros(9)),
    lambda: int8.quantize_rows(torch.zeros(9, 0)),
    lambda: int8.quantize_rows(torch.zeros(2, 2 ** 17 + 1, **META)),
    lambda: int8.quantize_rows(torch.zeros(2 ** 25 + 1, 2, **META)),
    lambda: int8.pack_rows(torch.zeros(9, 16), torch.zeros(9)),
    lambda: int8.pack_rows(torch.zeros(9, 16, dtype=torch.int8), torch.zeros(8)),
    lambda: int8.pack_rows(torch.zeros(9, 16, dtype=torch.int8), torch.zeros(9, dtype=torch.int32)),
    lambda: int8.pack_rows(torch.zeros(9, 16, dtype=torch.int8), torch.zeros(9, **META)),
    lambda: int8.dequantize((H, H)),
    lambda: int8.dequantize(rows(shape=(9, 80))),
    lambda: int8.dequantize(rows(shape=(300, 16))),
    lambda: int8.dequantize(rows(scale=torch.zeros(8))),
    lambda: int8.dequantize(rows(scale=torch.zeros(9, dtype=torch.float64))),
    lambda: int8.dequantize(rows(scale=torch.zeros(18)[::2])),
    lambda: int8.head_logits(H, H),
    lambda: int8.head_logits(torch.zeros(4, 15), rows()),
    lambda: int8.head_logits(torch.zeros(()), rows()),
    lambda: int8.head_logits(H, rows(), torch.zeros(8)),
    lambda: int8.head_logits(H, rows(), torch.zeros(9, dtype=torch.int32)),
    lambda: int8.head_logits(H, rows(device="meta")),
    lambda: int8.head_logits(H, rows(), torch.zeros(9, **META)),
    lambda: int8.head_logits(H.clone().requires_grad_(True), rows()),
    lambda: int8.head_logits(H, rows(), torch.zeros(9, requires_grad=True)),
])
def test_value_errors(call):
    with pytest.raises(ValueError):
        call()


@pytest.mark.parametrize("call", [
    lambda: swvr_amd.select_beams(X.double(), S),
    lambda: int8.quantize_rows(H.double()),
    lambda: int8.head_logits(H.double(), rows()),
    lambda: int8.head_logits(H, rows(), dtype=torch.float64),
])
def test_unsupported_types(call):
    with pytest.raises(NotImplementedError):
        call()


@pytest.mark.parametrize("call", [
    lambda: swvr_amd.select_beams(X, S),
    lambda: swvr_amd.reorder_beams(C, P),
    lambda: swvr_amd.reorder_beams(C, P, inplace=True),
    lambda: int8.quantize_rows(H),
    lambda: int8.pack_rows(torch.zeros(9, 16, dtype=torch.int8), torch.zeros(9)),
    lambda: int8.dequantize(rows()),
    lambda: int8.head_logits(H, rows()),
])
def test_cpu_tensors_are_refused(call):
    with pytest.raises(RuntimeError, match="AMD GPUs"):
        call()


def test_meta_tensors_give_shapes():
    x, s = torch.zeros(2, 5, 3, 9, dtype=torch.bfloat16, **META), torch.zeros(2, 5, 3, dtype=torch.float64, **META)
    token, parent, score = swvr_amd.select_beams(x, s, 6)
    assert token.shape == parent.shape == score.shape == (2, 5, 6)
    assert token.dtype == parent.dtype == torch.int64 and score.dtype == torch.float64
    assert swvr_amd.select_beams(x, s.to(torch.float16))[2].dtype == torch.float32
    c = torch.zeros(2, 5, 3, 7, 8, dtype=torch.int8, **META)
    assert swvr_amd.reorder_beams(c, parent).shape == (2, 5, 6, 7, 8)
    assert swvr_amd.reorder_beams([c], parent[..., :3], inplace=True)[0] is c
    cache = collections.namedtuple("Cache", "k v")(c, c.float())
    moved = swvr_amd.reorder_beams(cache, parent)
    assert type(moved) is type(cache) and moved.k.shape == moved.v.shape == (2, 5, 6, 7, 8) and moved.v.dtype == torch.float32
    assert swvr_amd.reorder_beams(cache, parent[..., :3], inplace=True) is cache
    w = int8.quantize_rows(torch.zeros(300, 100, **META))
    assert w.q.shape == (16, 2, 2048) and w.scale.shape == (300,) and w.shape == (300, 100)
    assert int8.dequantize(w).shape == (300, 100)
    out = int8.head_logits(torch.zeros(2, 4, 100, dtype=torch.float16, **META), w)
    assert out.shape == (2, 4, 300) and out.dtype == torch.float16
    assert int8.pack_rows(torch.zeros(300, 100, dtype=torch.int8, **META), torch.zeros(300, **META)).q.shape == (16, 2, 2048)


def test_geometry_of_states():
    g = lambda x, nb=1: _geometry(x.shape, x.stride(), x.element_size(), nb)
    x = torch.zeros(2, 3, 4, 10, 8, dtype=torch.float16)
    assert g(x) == (4 * 10 * 8 * 2, 1, 1, (3 * 4 * 10 * 8 * 2, 4 * 10 * 8 * 2, 0, 0), (0, 0))
    part = x[:, :, :, :7]     # dense pieces of 7 x 8, 4 of them
    assert g(part) == (7 * 8 * 2, 4, 1, (1920, 640, 0, 160), (0, 112))
    assert g(x[..., :5]) == (10, 40, 1, (1920, 640, 0, 16), (0, 10))
    assert g(x[:, :, :, :7, :5]) == (10, 7, 4, (1920, 640, 160, 16), (70, 10))
    assert g(x[..., ::2]) == (2, 160, 1, (1920, 640, 0, 4), (0, 2))
    assert g(x[:, :, ::2, ::3, ::2]) is None
    big = torch.zeros(2, 3, 2 ** 16, 2 ** 16, device="meta", dtype=torch.uint8)   # 4 GB a beam: in one piece alone
    assert g(big) == (2 ** 32, 1, 1, (3 * 2 ** 32, 2 ** 32, 0, 0), (0, 0)) and g(big[..., 1:]) is not None
    assert g(torch.zeros(2, 3, 2 ** 17, 2 ** 16, device="meta", dtype=torch.uint8)[..., 1:]) is None
    y = torch.zeros(2, 3, 4, 8)
    assert g(y, 2) == (32, 1, 1, (128, 32, 0, 0), (0, 0))
    assert g(y[:, :2], 2) is None           # leading dimensions apart
    assert g(torch.zeros(4, 8), 0) == (32, 1, 1, (0, 32, 0, 0), (0, 0))
    assert g(torch.zeros(3, 1, 1)) == (4, 1, 1, (4, 0, 0, 0), (0, 0))


def test_views_with_shared_elements():
    f = lambda x: _overlaps(x.shape, x.stride())
    x = torch.zeros(2, 3, 4)
    assert not f(x) and not f(x.transpose(0, 2)) and not f(x[:, ::2]) and not f(x[:1])
    assert f(x[:, :1].expand(2, 3, 4)) and f(torch.zeros(20).as_strided((2, 3, 4), (8, 2, 1)))


A = ctypes.c_void_p(4096)


def select(dtype=_lib.BF16, B=2, W=3, V=8, k=3, logits=A, ld=8, scores=A, s64=0, finished=None, end=0, lengths=None,
           alpha=0.0, token=A, parent=A, score=A, ws=A, nbytes=1 << 30):
    return _lib.load().swvr_select_beams(dtype, B, W, V, k, logits, ld, scores, s64, finished, end, lengths, alpha, token,
                                         parent, score, ws, nbytes, None)


def reorder(n=1, src=(4096,), dst=(8192,), B=2, W=3, k=3, parents=A, id64=1, run=8, n1=1, n2=1, steps=(24, 8, 0, 0), to=(24, 8, 0, 0)):
    at = lambda xs: (ctypes.c_void_p * len(xs))(*xs) if xs is not None else None
    st = lambda xs: (ctypes.c_int64 * 4)(*xs) if xs is not None else None
    return _lib.load().swvr_reorder_beams(n, at(src), at(dst), B, W, k, parents, id64, run, n1, n2, st(steps), st(to), None)


def quantize(dtype=_lib.BF16, R=4, K=16, x=A, ld=16, image=A, scale=A):
    return _lib.load().swvr_int8_quantize(dtype, R, K, x, ld, image, scale, None)


def pack(R=4, K=16, q=A, ld=16, image=A):
    return _lib.load().swvr_int8_pack(R, K, q, ld, image, None)


def unpack(R=4, K=16, image=A, scale=A, out=A):
    return _lib.load().swvr_int8_unpack(R, K, image, scale, out, None)


def logits(dtype=_lib.BF16, out_dtype=_lib.BF16, N=4, K=16, V=9, h=A, ldh=16, image=A, scale=A, bias=None, b=0, out=A, ws=A,
           nbytes=1 << 40):
    return _lib.load().swvr_int8_logits(dtype, out_dtype, N, K, V, h, ldh, image, scale, bias, b, 1.0, out, ws, nbytes, None)


@pytest.mark.parametrize("fn,kw,code", [
    (select, dict(dtype=_lib.F64), _lib.EDTYPE),
    (select, dict(B=-1), _lib.EINVAL),
    (select, dict(W=0), _lib.EINVAL),
    (select, dict(W=257), _lib.EINVAL),
    (select, dict(k=0), _lib.EINVAL),
    (select, dict(k=257), _lib.EINVAL),
    (select, dict(V=0), _lib.EINVAL),
    (select, dict(V=2 ** 21 + 1), _lib.EINVAL),
    (select, dict(B=2 ** 23 + 1, W=1), _lib.EINVAL),
    (select, dict(B=2 ** 23, W=2), _lib.EINVAL),
    (select, dict(B=2 ** 16, W=8, V=2 ** 18), _lib.EINVAL),
    (select, dict(ld=-1), _lib.EINVAL),
    (select, dict(s64=2), _lib.EINVAL),
    (select, dict(finished=A, end=8), _lib.EINVAL),
    (select, dict(finished=A, end=-1), _lib.EINVAL),
    (select, dict(alpha=-1.0), _lib.EINVAL),
    (select, dict(alpha=17.0), _lib.EINVAL),
    (select, dict(alpha=float("nan")), _lib.EINVAL),
    (select, dict(logits=None), _lib.EINVAL),
    (select, dict(logits=ctypes.c_void_p(4097)), _lib.EINVAL),
    (select, dict(scores=None), _lib.EINVAL),
    (select, dict(parent=None), _lib.EINVAL),
    (select, dict(ws=None), _lib.EWORKSPACE),
    (select, dict(ws=ctypes.c_void_p(4104)), _lib.EWORKSPACE),
    (select, dict(nbytes=16), _lib.EWORKSPACE),
    (reorder, dict(n=-1), _lib.EINVAL),
    (reorder, dict(B=-1), _lib.EINVAL),
    (reorder, dict(W=0), _lib.EINVAL),
    (reorder, dict(W=257), _lib.EINVAL),
    (reorder, dict(k=257), _lib.EINVAL),
    (reorder, dict(run=-8), _lib.EINVAL),
    (reorder, dict(run=2 ** 41), _lib.EINVAL),
    (reorder, dict(run=2 ** 30, n1=2 ** 30, n2=2 ** 30), _lib.EINVAL),
    (reorder, dict(run=2 ** 20, n1=2 ** 6, n2=2 ** 6), _lib.EINVAL),
    (reorder, dict(id64=2), _lib.EINVAL),
    (reorder, dict(dst=None, k=4), _lib.EINVAL),
    (reorder, dict(dst=None, W=65, k=65), _lib.EINVAL),
    (reorder, dict(src=None), _lib.EINVAL),
    (reorder, dict(src=(0,)), _lib.EINVAL),
    (reorder, dict(dst=(0,)), _lib.EINVAL),
    (reorder, dict(parents=None), _lib.EINVAL),
    (reorder, dict(steps=None), _lib.EINVAL),
    (reorder, dict(to=None), _lib.EINVAL),
    (reorder, dict(steps=(24, -8, 0, 0)), _lib.EINVAL),
    (quantize, dict(dtype=_lib.F64), _lib.EDTYPE),
    (quantize, dict(R=-1), _lib.EINVAL),
    (quantize, dict(R=2 ** 25 + 1), _lib.EINVAL),
    (quantize, dict(K=0), _lib.EINVAL),
    (quantize, dict(K=2 ** 17 + 1), _lib.EINVAL),
    (quantize, dict(ld=-1), _lib.EINVAL),
    (quantize, dict(x=None), _lib.EINVAL),
    (quantize, dict(x=ctypes.c_void_p(4097)), _lib.EINVAL),
    (quantize, dict(image=ctypes.c_void_p(4104)), _lib.EINVAL),
    (quantize, dict(scale=None), _lib.EINVAL),
    (pack, dict(K=0), _lib.EINVAL),
    (pack, dict(ld=-1), _lib.EINVAL),
    (pack, dict(q=None), _lib.EINVAL),
    (unpack, dict(R=-1), _lib.EINVAL),
    (unpack, dict(R=2 ** 25, K=4097), _lib.EINVAL),
    (unpack, dict(scale=None), _lib.EINVAL),
    (unpack, dict(out=ctypes.c_void_p(4100)), _lib.EINVAL),
    (logits, dict(dtype=_lib.F64), _lib.EDTYPE),
    (logits, dict(out_dtype=3), _lib.EDTYPE),
    (logits, dict(bias=A, b=4), _lib.EDTYPE),
    (logits, dict(N=-1), _lib.EINVAL),
    (logits, dict(N=2 ** 24 + 1), _lib.EINVAL),
    (logits, dict(N=2 ** 24, V=2 ** 20), _lib.EINVAL),
    (logits, dict(V=-1), _lib.EINVAL),
    (logits, dict(K=0), _lib.EINVAL),
    (logits, dict(ldh=-1), _lib.EINVAL),
    (logits, dict(h=None), _lib.EINVAL),
    (logits, dict(image=ctypes.c_void_p(4104)), _lib.EINVAL),
    (logits, dict(scale=None), _lib.EINVAL),
    (logits, dict(out=None), _lib.EINVAL),
    (logits, dict(ws=None), _lib.EWORKSPACE),
    (logits, dict(nbytes=64), _lib.EWORKSPACE),
])
def test_abi_refusals(fn, kw, code):
    assert fn(**kw) == code
    assert _lib.load().swvr_last_error()


def test_abi_empty_calls_launch_nothing():
    assert select(B=0, logits=None, scores=None, token=None, ws=None) == _lib.OK
    assert reorder(n=0, src=None, dst=(8192,)) == _lib.OK
    assert reorder(B=0, src=(0,)) == _lib.OK
    assert reorder(run=0, parents=None) == _lib.OK
    assert quantize(R=0, x=None, image=None, scale=None) == _lib.OK
    assert pack(R=0, q=None, image=None) == _lib.OK
    assert unpack(R=0, image=None, scale=None, out=None) == _lib.OK
    assert logits(N=0, h=None, out=None, ws=None) == _lib.OK
    assert logits(V=0, image=None, out=None, ws=None) == _lib.OK


def test_sizes():
    lib = _lib.load()
    assert lib.swvr_int8_size(300, 100) == 16 * 2 * 2048 and lib.swvr_int8_size(0, 5) == 0 and lib.swvr_int8_size(5, 0) == 0
    assert lib.swvr_int8_logits_workspace_size(300, 100) == 1280 + 16 * 2 * 2048
    assert lib.swvr_select_beams_workspace_size(2, 257, 9, 1) == 0
    # of 6 rows of 5000 logits: 3 sub-blocks of 16 groups, 4 candidates
    assert lib.swvr_select_beams_workspace_size(2, 3, 5000, 4) == 6 * 3 * (8 + 4 + 16 * 4) + 6 * 4 * 2 * 8 + 6 * 4 * 4 + 6 * 4
