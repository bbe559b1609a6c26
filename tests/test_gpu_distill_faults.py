"""softmax_distill where its inputs are at fault: ids outside the vocabulary and NaN must show in the loss and in every
gradient that their token reaches, and in nothing else; and at the ends of its inputs' ranges, where nothing may be
lost."""
import math

import pytest
import torch

import swvr_amd
from swvr_amd import _lib

from .test_gpu_distill import close, formula

pytestmark = pytest.mark.gpu
DEV = "cuda"
DTYPES = [torch.bfloat16, torch.float16, torch.float32]
N, K, V, T, BAD = 40, 512, 300, 5, 7


def make(dtype, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    r = lambda *s, sc=1.0: (sc * torch.randn(*s, device=DEV, generator=g)).to(dtype)
    ids = torch.randint(0, V, (N, T), device=DEV, generator=g)
    return r(N, K), r(V, K, sc=2 * K ** -0.5), r(V, sc=0.5), torch.randn(N, T, device=DEV, generator=g), ids


def step(h, W, b, t, ids, reduction, g=None, **kw):
    """(loss, gh, gW, gb) of one call."""
    xs = [x.detach().requires_grad_(True) for x in (h, W, b)]
    loss = swvr_amd.softmax_distill(xs[0], xs[1], t, ids, xs[2], reduction=reduction, **kw)
    return (loss.detach(), *torch.autograd.grad(loss, xs, torch.ones_like(loss) if g is None else g))


def spoil(how, t, ids):
    t, ids = t.clone(), ids.clone()
    if how == "id":
        ids[BAD, 2] = V
    elif how == "id past 32 bits":
        ids[BAD, 2] = 2 ** 32 + 5          # 5, if it were cut
    elif how == "improbable id":           # e^-300 is 0 in fp32
        t[BAD, 2], ids[BAD, 2] = t[BAD].max() - 300, V
    else:
        t[BAD, 2] = math.nan
    return t, ids


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("how", ["id", "id past 32 bits", "improbable id", "nan"])
@pytest.mark.parametrize("reduction", ["none", "sum", "mean"])
@pytest.mark.parametrize("chunk", [None, 128])   # scores kept, and formed again in three chunks
def test_a_token_at_fault_shows_in_its_gradients(dtype, how, reduction, chunk):
    tag = _lib.DTYPE_TAG[dtype]
    assert _lib.load().swvr_distill_scores_size(tag, tag, N, K, V, K) > 0
    h, W, b, t, ids = make(dtype)
    good = step(h, W, b, t, ids, reduction, chunk_size=chunk)
    loss, gh, gW, gb = step(h, W, b, *spoil(how, t, ids), reduction, chunk_size=chunk)
    rest = torch.arange(N, device=DEV) != BAD
    if reduction == "none":
        assert loss[BAD].isnan() and torch.equal(loss[rest], good[0][rest])
    else:
        assert loss.isnan()
    assert gh[BAD].isnan().all() and torch.equal(gh[rest], good[1][rest])
    assert gW.isnan().all() and gb.isnan().all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("chunk", [None, 128])
def test_a_token_at_fault_that_nothing_asks_for(dtype, chunk):
    """Its term left out of what is differentiated, or its weight zero: the gradients of the others."""
    h, W, b, t, ids = make(dtype)
    t2, ids2 = spoil("id", t, ids)
    t2[BAD, 0] = math.nan
    keep = torch.ones(N, device=DEV)
    keep[BAD] = 0
    want = step(h, W, b, t, ids, "none", g=keep, chunk_size=chunk)
    got = step(h, W, b, t2, ids2, "none", g=keep, chunk_size=chunk)
    assert got[0][BAD].isnan()
    for a, c in zip(got[1:], want[1:]):
        assert torch.equal(a, c) and torch.isfinite(a).all()
    for a, c in zip(step(h, W, b, t2, ids2, "mean", weight=keep, chunk_size=chunk),
                    step(h, W, b, t, ids, "mean", weight=keep, chunk_size=chunk)):
        assert torch.equal(a, c) and torch.isfinite(a).all()


@pytest.mark.parametrize("t_dtype", DTYPES)
@pytest.mark.parametrize("tau", [1.0, 0.5, 0.01])
@pytest.mark.parametrize("many", [1, 20])       # lists within a wave's 64 entries, and longer ones
def test_teachers_of_lowest_and_highest_values(t_dtype, tau, many):
    """Finite logits, however low, are entries: a list of nothing else is uniform at every temperature."""
    h, W, b, _, ids = make(torch.float32)
    ids = ids.repeat(1, many)
    low, top = torch.finfo(t_dtype).min, torch.finfo(t_dtype).max
    t = torch.zeros(N, T * many, device=DEV, dtype=t_dtype)
    t[::8] = low
    t[1::8] = low
    t[1::8, 3] = 0
    t[2::8] = top
    t[3::8, 0], t[3::8, 1:] = top, low
    t[4::8, ::2], t[4::8, 1::2] = low, -math.inf
    t[5::8, ::2], t[5::8, 1::2] = -math.inf, top
    t[6::8] = -math.inf
    # the softmax's probabilities underflow at low temperatures: those below fp32's smallest normal number, 2^-126, may
    # come as 0, so an element of dS is off by that much more (its cotangent is 1 or less, its LSE term 0), and a
    # gradient by the sum of it times what the element is multiplied by
    f = 2.0 ** -126 / tau
    floor = dict(h=f * W.double().abs().sum(dim=0), W=f * h.double().abs().sum(dim=0), b=f * N)
    for reduction in ("none", "mean"):
        loss, *grads = step(h, W, b, t, ids, reduction, temperature=tau)
        want, want_g, tol = formula(h, W, b, t, ids, tau=tau, reduction=reduction)
        close(loss, want, tol["loss"])
        for name, got in zip("hWb", grads):
            close(got, want_g[name], tol[name] + floor[name])
        if reduction == "none":
            assert (loss[6::8] == 0).all() and (loss[::8] != 0).all()
        assert (grads[0][6::8] == 0).all() and (grads[0][::8] != 0).any(dim=1).all()


@pytest.mark.parametrize("dtype,K", [(torch.bfloat16, 1024), (torch.float16, 1024), (torch.float32, 256)])
@pytest.mark.parametrize("reduction", ["none", "mean"])
@pytest.mark.parametrize("chunk", [None, 128])
def test_dropped_tokens_may_hold_anything_where_scores_are_kept(dtype, K, reduction, chunk):
    """A forward that keeps the scores computes the dropped tokens' too; token 0, whose scores padding reads, among them."""
    n, tag = 70, _lib.DTYPE_TAG[dtype]
    assert _lib.load().swvr_distill_scores_size(tag, tag, n, K, V, K) > 0
    g = torch.Generator(device=DEV).manual_seed(K)
    h = torch.randn(n, K, device=DEV, generator=g).to(dtype)
    W = (2 * K ** -0.5 * torch.randn(V, K, device=DEV, generator=g)).to(dtype)
    b = torch.randn(V, device=DEV, generator=g).to(dtype)
    t, ids = torch.randn(n, T, device=DEV, generator=g), torch.randint(0, V, (n, T), device=DEV, generator=g)
    weight = torch.ones(n, device=DEV)
    weight[::4] = 0
    want = step(h, W, b, t, ids, reduction, weight=weight, chunk_size=chunk)
    h2, t2, ids2 = h.clone(), t.clone(), ids.clone()
    h2[::8], h2[4::8] = math.nan, math.inf
    t2[::4], ids2[::4] = math.nan, 10 ** 9
    for a, c in zip(step(h2, W, b, t2, ids2, reduction, weight=weight, chunk_size=chunk), want):
        assert torch.equal(a, c) and torch.isfinite(a).all()
    # dropped by having no entries
    ids3 = ids2.clone()
    ids3[::4] = -1
    for a, c in zip(step(h2, W, b, t2, ids3, reduction, chunk_size=chunk), want):
        assert torch.equal(a, c)
