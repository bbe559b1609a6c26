"""Host-side checks of the token operators that need no GPU: refused arguments, shapes under tracing, and the
C ABI's own checks (nothing is launched)."""
import ctypes

import pytest
import torch

import swvr_amd
from swvr_amd import _lib

H, W, B = torch.zeros(4, 16), torch.zeros(9, 16), torch.zeros(9)
T, I = torch.zeros(4, 3), torch.zeros(4, 3, dtype=torch.int64)
LOGITS, U = torch.zeros(4, 9), torch.zeros(4)


def distill(h=H, w=W, t=T, i=I, b=B, **kw):
    return swvr_amd.softmax_distill(h, w, t, i, b, **kw)


@pytest.mark.parametrize("call", [
    lambda: distill(w=torch.zeros(16)),
    lambda: distill(w=torch.zeros(0, 16), b=None),
    lambda: distill(w=torch.zeros(9, 15)),
    lambda: distill(b=torch.zeros(8)),
    lambda: distill(t=torch.zeros(4, 2)),
    lambda: distill(t=torch.zeros(3, 3), i=I[:3]),
    lambda: distill(t=torch.zeros(4, 0), i=I[:, :0]),
    lambda: distill(t=torch.zeros(4, 1025), i=torch.zeros(4, 1025, dtype=torch.int64)),
    lambda: distill(i=I.float()),
    lambda: distill(i=I.bool()),
    lambda: distill(t=T.long()),
    lambda: distill(weight=torch.zeros(3)),
    lambda: distill(weight=torch.zeros(4, requires_grad=True)),
    lambda: distill(t=T.clone().requires_grad_(True)),
    lambda: distill(temperature=0.0),
    lambda: distill(temperature=-1.0),
    lambda: distill(temperature=float("nan")),
    lambda: distill(temperature=float("inf")),
    lambda: distill(reduction="avg"),
    lambda: distill(chunk_size=-3),
    lambda: swvr_amd.embedding_lookup(I, torch.zeros(9)),
    lambda: swvr_amd.embedding_lookup(I.float(), W),
    lambda: swvr_amd.embedding_lookup(I.bool(), W),
    lambda: swvr_amd.sample_tokens(torch.zeros(4, 0), U),
    lambda: swvr_amd.sample_tokens(torch.zeros(()), U),
    lambda: swvr_amd.sample_tokens(LOGITS, U[:3]),
    lambda: swvr_amd.sample_tokens(LOGITS, U.long()),
    lambda: swvr_amd.sample_tokens(LOGITS, U, temperature=-0.5),
    lambda: swvr_amd.sample_tokens(LOGITS, U, temperature=float("inf")),
    lambda: swvr_amd.sample_tokens(LOGITS, U, temperature=float("nan")),
    lambda: swvr_amd.sample_tokens(LOGITS, U, top_k=-1),
    lambda: swvr_amd.sample_tokens(LOGITS, U, top_p=1.5),
    lambda: swvr_amd.sample_tokens(LOGITS, U, top_p=float("nan")),
    lambda: swvr_amd.sample_tokens(LOGITS, U, min_p=-0.1),
    lambda: swvr_amd.sample_tokens(LOGITS, U, min_p=1.1),
    lambda: swvr_amd.sample_tokens(LOGITS, U, top_k=torch.zeros(3, dtype=torch.int32)),
    lambda: swvr_amd.sample_tokens(LOGITS, U, top_k=torch.zeros(4)),
    lambda: swvr_amd.sample_tokens(LOGITS, U, temperature=torch.zeros(())),
])
def test_value_errors(call):
    with pytest.raises(ValueError):
        call()


@pytest.mark.parametrize("call", [
    lambda: distill(h=H.double(), w=W.double()),
    lambda: swvr_amd.embedding_lookup(I, W.to(torch.complex64)),
    lambda: swvr_amd.embedding_lookup(I, W.to(torch.int8)),
    lambda: swvr_amd.sample_tokens(LOGITS.double(), U),
])
def test_unsupported_types(call):
    with pytest.raises(NotImplementedError):
        call()


@pytest.mark.parametrize("call", [
    lambda: distill(),
    lambda: swvr_amd.embedding_lookup(I, W),
    lambda: swvr_amd.sample_tokens(LOGITS, U),
])
def test_cpu_tensors_are_refused(call):
    with pytest.raises(RuntimeError, match="AMD GPUs"):
        call()


def test_tensors_on_two_devices_are_refused():
    meta = torch.zeros(9, 16, device="meta")
    with pytest.raises(ValueError):
        distill(w=meta)
    with pytest.raises(ValueError):
        swvr_amd.embedding_lookup(I, meta)
    with pytest.raises(ValueError):
        swvr_amd.sample_tokens(torch.zeros(4, 9, device="meta"), U)
    with pytest.raises(ValueError):
        swvr_amd.sample_tokens(LOGITS, U, top_p=torch.zeros(4, device="meta"))


def test_meta_tensors_give_shapes_and_gradients():
    m = dict(device="meta")
    h, w, b = (torch.zeros(*s, dtype=torch.bfloat16, **m).requires_grad_(True) for s in ((2, 5, 16), (9, 16), (9,)))
    t, i = torch.zeros(2, 5, 3, **m), torch.zeros(2, 5, 3, dtype=torch.int64, **m)
    loss = swvr_amd.softmax_distill(h, w, t, i, b)
    assert loss.shape == () and loss.dtype == torch.float32
    assert [g.shape for g in torch.autograd.grad(loss, (h, w, b))] == [h.shape, w.shape, b.shape]
    assert swvr_amd.softmax_distill(h, w, t, i, b, reduction="none").shape == (2, 5)
    out = swvr_amd.embedding_lookup(i, w)
    assert out.shape == (2, 5, 3, 16) and out.dtype == torch.bfloat16
    assert torch.autograd.grad(out.sum(), w)[0].shape == w.shape
    token, logprob = swvr_amd.sample_tokens(torch.zeros(2, 5, 9, **m), torch.zeros(2, 5, **m))
    assert token.shape == logprob.shape == (2, 5)
    assert token.dtype == torch.int64 and logprob.dtype == torch.float32


P = ctypes.c_void_p(16)


def embedding(dtype=_lib.BF16, id64=1, N=4, V=8, D=4, ids=P, E=P, lde=4, out=P):
    return _lib.load().swvr_embedding(dtype, id64, N, V, D, ids, E, lde, 1.0, out, None, None)


def embedding_bwd(dtype=_lib.BF16, id64=1, N=4000, V=8, D=4, ids=P, g=P, ldg=4, gE=P, ws=P, nbytes=1 << 20):
    return _lib.load().swvr_embedding_bwd(dtype, id64, N, V, D, ids, g, ldg, 1.0, None, gE, ws, nbytes, None)


def sample(dtype=_lib.BF16, R=4, V=8, logits=P, ld=8, u=P, u64=0, tau=1.0, token=P, logprob=P, ws=P, nbytes=1 << 30):
    return _lib.load().swvr_sample(dtype, R, V, logits, ld, u, u64, tau, None, 0, None, 1.0, None, 0.0, None, token,
                                   logprob, ws, nbytes, None)


def distill_abi(dtype=_lib.BF16, N=4, K=16, V=8, T=2, h=P, ids=P, id64=1, teacher=P, t_dtype=_lib.F32, tau=1.0, red=2,
                out=P, c=P, lse=P, p=P, q=P, coef=P, scores=None, ws=P, nbytes=1 << 30):
    return _lib.load().swvr_distill(dtype, dtype, dtype, N, K, V, T, h, 16, P, 16, None, 0, None, 1.0, ids, id64, T, teacher,
                                    t_dtype, T, tau, None, 0.0, red, out, c, lse, p, q, coef, scores, ws, nbytes, None)


def distill_bwd_abi(dtype=_lib.BF16, N=4, V=8, T=2, tau=1.0, chunk=8192, g=P, gb=None, scores=None, ws=P, nbytes=1 << 30):
    return _lib.load().swvr_distill_bwd(dtype, dtype, dtype, N, 16, V, T, P, 16, P, 16, None, 1.0, P, 1, T, tau, 0.0, 2,
                                        g, P, P, P, P, P, scores, chunk, P, dtype, P, dtype, gb, 2, ws, nbytes, None)


@pytest.mark.parametrize("fn,kw,code", [
    (embedding, dict(dtype=3), _lib.EDTYPE),
    (embedding, dict(id64=2), _lib.EINVAL),
    (embedding, dict(N=-1), _lib.EINVAL),
    (embedding, dict(N=2 ** 31), _lib.EINVAL),
    (embedding, dict(V=2 ** 31 - 1), _lib.EINVAL),
    (embedding, dict(lde=3), _lib.EINVAL),
    (embedding, dict(ids=None), _lib.EINVAL),
    (embedding, dict(E=None), _lib.EINVAL),
    (embedding, dict(out=None), _lib.EINVAL),
    (embedding_bwd, dict(dtype=9), _lib.EDTYPE),
    (embedding_bwd, dict(g=None), _lib.EINVAL),
    (embedding_bwd, dict(gE=None), _lib.EINVAL),
    (embedding_bwd, dict(ldg=-4), _lib.EINVAL),
    (embedding_bwd, dict(ws=None), _lib.EWORKSPACE),
    (embedding_bwd, dict(nbytes=16), _lib.EWORKSPACE),
    (sample, dict(dtype=_lib.F64), _lib.EDTYPE),
    (sample, dict(V=0), _lib.EINVAL),
    (sample, dict(R=-1), _lib.EINVAL),
    (sample, dict(ld=-1), _lib.EINVAL),
    (sample, dict(u64=5), _lib.EINVAL),
    (sample, dict(tau=-1.0), _lib.EINVAL),
    (sample, dict(tau=float("nan")), _lib.EINVAL),
    (sample, dict(logits=ctypes.c_void_p(17)), _lib.EINVAL),
    (sample, dict(token=None), _lib.EINVAL),
    (sample, dict(V=50000, nbytes=1000), _lib.EWORKSPACE),
    (sample, dict(V=50000, ws=None), _lib.EWORKSPACE),
    (distill_abi, dict(dtype=_lib.F64), _lib.EDTYPE),
    (distill_abi, dict(t_dtype=5), _lib.EDTYPE),
    (distill_abi, dict(T=0), _lib.EINVAL),
    (distill_abi, dict(T=1025), _lib.EINVAL),
    (distill_abi, dict(N=2 ** 30, T=4), _lib.EINVAL),
    (distill_abi, dict(tau=0.0), _lib.EINVAL),
    (distill_abi, dict(red=3), _lib.EINVAL),
    (distill_abi, dict(ids=None), _lib.EINVAL),
    (distill_abi, dict(teacher=None), _lib.EINVAL),
    (distill_abi, dict(lse=None), _lib.EINVAL),
    (distill_abi, dict(out=None), _lib.EINVAL),
    (distill_abi, dict(c=None), _lib.EINVAL),
    (distill_abi, dict(q=None), _lib.EINVAL),
    (distill_abi, dict(K=12), _lib.EINVAL),
    (distill_abi, dict(h=ctypes.c_void_p(8)), _lib.EINVAL),
    (distill_abi, dict(nbytes=64), _lib.EWORKSPACE),
    (distill_abi, dict(N=1000, V=4000, scores=P), _lib.EINVAL),       # more tokens than scores are kept of
    (distill_bwd_abi, dict(N=1000, V=4000, scores=P), _lib.EINVAL),
    (distill_bwd_abi, dict(dtype=7), _lib.EDTYPE),
    (distill_bwd_abi, dict(chunk=0), _lib.EINVAL),
    (distill_bwd_abi, dict(g=None), _lib.EINVAL),
    (distill_bwd_abi, dict(gb=P), _lib.EINVAL),
    (distill_bwd_abi, dict(ws=None), _lib.EWORKSPACE),
    (distill_bwd_abi, dict(nbytes=64), _lib.EWORKSPACE),
])
def test_abi_refusals(fn, kw, code):
    assert fn(**kw) == code
    assert _lib.load().swvr_last_error()


@pytest.mark.parametrize("bias_dtype,tau", [(_lib.BF16, 1.0), (_lib.F32, 2.0)])
def test_abi_refuses_a_bias_as_its_own_scaled_copy(bias_dtype, tau):
    lib = _lib.load()
    assert lib.swvr_distill(_lib.BF16, _lib.BF16, _lib.BF16, 4, 16, 8, 2, P, 16, P, 16, P, bias_dtype, P, 1.0, P, 1, 2, P,
                            _lib.F32, 2, tau, None, 0.0, 2, P, P, P, P, P, P, None, P, 1 << 30, None) == _lib.EINVAL
    assert b"temperature 1" in lib.swvr_last_error()


def test_abi_empty_calls_launch_nothing():
    assert embedding(N=0, ids=None, out=None) == _lib.OK
    assert embedding(D=0, lde=0, E=None, out=None) == _lib.OK
    assert embedding_bwd(V=0, gE=None) == _lib.OK
    assert sample(R=0, logits=None, u=None, token=None, logprob=None) == _lib.OK
