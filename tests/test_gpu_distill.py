"""softmax_distill on the GPU against its formula in 64 bits on the operands as the kernels get them, with
tolerances from the arithmetic, element by element.

With u = 2^-24 (half a step of fp32) and r half a step of the compute dtype:
  a score is a dot product of K fp32 products and a sum with the bias: off by dS <= (K + 4) u (|h| |W|^T s / tau +
    |b| / tau); LSE by the largest dS of its row and the rounding of its own sums, in exponentials good to 2^-21 each and
    2 u |LSE|;
  softmax at a score is off by (dS + dLSE + 2^-21 (1 + |S - LSE|)) of itself, the teacher's p by 2^-21;
  an element of dS is staged rounded to the compute dtype (r of itself; fp16 below its normal numbers by 2^-25);
  a gradient sums those errors times |W| or |h|, its own fp32 sums (n u of the magnitudes) and its rounding."""
import math

import pytest
import torch

import swvr_amd

from .gpu_util import rel_err

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: U}
TINY = {torch.bfloat16: 0.0, torch.float16: 2.0 ** -25, torch.float32: 0.0}


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def make(N, K, V, T, dtype, seed=0, bias=True, absent=0.2, spread=2.0):
    g = gen(seed)
    r = lambda *s, sc=1.0: (sc * torch.randn(*s, device=DEV, generator=g)).to(dtype)
    h, W = r(N, K), r(V, K, sc=spread * K ** -0.5)
    b = r(V, sc=0.5) if bias else None
    ids = torch.randint(0, V, (N, T), device=DEV, generator=g)
    ids = torch.where(torch.rand(N, T, device=DEV, generator=g) < absent, -1, ids)
    t = 3 * torch.randn(N, T, device=DEV, generator=g)
    return h, W, b, t, ids


def formula(h, W, b, t, ids, tau=1.0, weight=None, z=0.0, reduction="mean", scale=1.0, g=None, cdt=None):
    """Everything in 64 bits: loss, gradients, and a dict of the elementwise tolerances of the gradients."""
    cdt = cdt or h.dtype
    out_t = dict(h=h.dtype, W=W.dtype, b=b.dtype if b is not None else None)
    hd, Wd = h.detach().to(cdt).double(), W.detach().to(cdt).double()
    bd = b.detach().double() if b is not None else torch.zeros(W.shape[0], dtype=torch.float64, device=DEV)
    N, K = hd.shape
    V, T = Wd.shape[0], ids.shape[1]
    S = (scale * hd @ Wd.t() + bd) / tau
    lse = torch.logsumexp(S, dim=1)
    td = t.double() / tau
    there = (ids >= 0) & (td != -math.inf)
    live = there.any(dim=1)
    td = torch.where(there, td, -math.inf)
    p = torch.where(live[:, None], torch.softmax(td, dim=1), 0.0).nan_to_num(0.0)
    logp = torch.where(p > 0, p.log(), 0.0)
    at = ids.long().clamp(0, V - 1)
    logq = S.gather(1, at) - lse[:, None]
    kl = torch.where(p > 0, p * (logp - logq), 0.0).sum(dim=1)
    w = weight.double() if weight is not None else torch.ones(N, dtype=torch.float64, device=DEV)
    w = torch.where(live, w, 0.0)
    term = torch.where(w != 0, w * (kl + z * lse.square()), 0.0)
    c = 1.0
    if reduction == "mean":
        c = 1.0 / w.sum() if w.sum() != 0 else 1.0
    loss = term if reduction == "none" else term.sum() * c
    gn = (g.double() if g is not None else 1.0) * w * c
    cn = gn * (1 + 2 * z * lse)
    P = torch.exp(S - lse[:, None])
    dense = torch.where(w[:, None] != 0, cn[:, None] * P, 0.0)
    sparse = torch.zeros_like(S).scatter_add_(1, at, torch.where(there, gn[:, None] * p, 0.0))
    dS = dense - sparse
    # tolerances
    mag = (abs(scale) * hd.abs() @ Wd.abs().t() + bd.abs()) / tau
    dScore = (K + 4) * U * mag
    dLse = dScore.amax(dim=1) + 2.0 ** -21 + 2 * U * lse.abs() + V * U * 0.5
    rel_q = dScore + dLse[:, None] + 2.0 ** -21 * (1 + (S - lse[:, None]).abs())
    e = dense.abs() * (rel_q + 4 * U) + sparse.abs() * (2.0 ** -20 + T * U)
    e = e + (dS.abs() + e) * HALF[cdt] + TINY[cdt]
    s = abs(scale) / tau
    tol = {}
    if out_t["h"] in HALF:
        want = scale / tau * dS @ Wd
        tol["h"] = s * (e @ Wd.abs() + (V + 8) * U * dS.abs() @ Wd.abs()) + want.abs() * HALF[out_t["h"]] + TINY[out_t["h"]]
    wantW = scale / tau * dS.t() @ hd
    tol["W"] = s * (e.t() @ hd.abs() + (N + 8) * U * dS.abs().t() @ hd.abs()) + wantW.abs() * HALF[out_t["W"]] + TINY[out_t["W"]]
    wantb = dS.sum(dim=0) / tau
    if b is not None:
        tol["b"] = ((e + (N + 8) * U * (dense.abs() + sparse.abs())).sum(dim=0) / tau + wantb.abs() * HALF[out_t["b"]]
                    + TINY[out_t["b"]])
    # the loss's terms: p's and the scores' errors times the magnitudes
    dterm = w.abs() * ((p * (dScore.gather(1, at) + dLse[:, None] + 2.0 ** -20 * (1 + logp.abs() + logq.abs()))).sum(dim=1)
                       + abs(z) * 2 * lse.abs() * dLse + (T + 8) * U * (kl.abs() + abs(z) * lse.square()))
    dterm = dterm.nan_to_num(0.0)
    tol["loss"] = dterm if reduction == "none" else dterm.sum() * abs(c) + (N + 8) * U * term.abs().sum() * abs(c)
    return loss, dict(h=want, W=wantW, b=wantb if b is not None else None), tol


def close(got, want, tol):
    assert got.shape == want.shape
    nan = torch.isnan(want)
    assert torch.equal(torch.isnan(got), nan)
    off = (got.double() - want).abs()
    assert not ((off > tol) & ~nan & (got.double() != want)).any(), (off - tol).max().item()


def check(h, W, b, t, ids, reduction="mean", weight=None, g=None, chunk_size=None, **kw):
    h, W = h.detach().requires_grad_(True), W.detach().requires_grad_(True)
    b = b.detach().requires_grad_(True) if b is not None else None
    loss = swvr_amd.softmax_distill(h, W, t, ids, b, weight=weight, reduction=reduction, chunk_size=chunk_size,
                                    temperature=kw.get("tau", 1.0), z_loss_weight=kw.get("z", 0.0),
                                    logit_scale=kw.get("scale", 1.0))
    assert loss.dtype == torch.float32
    xs = [x for x in (h, W, b) if x is not None]
    grads = torch.autograd.grad(loss, xs, g if g is not None else torch.ones_like(loss))
    want, want_g, tol = formula(h, W, b, t, ids, weight=weight, reduction=reduction, g=g, **kw)
    close(loss.detach(), want, tol["loss"])
    for name, x, got in zip("hWb", xs, grads):
        assert got.dtype == x.dtype
        close(got, want_g[name], tol[name])
    with torch.no_grad():
        same = swvr_amd.softmax_distill(h, W, t, ids, b, weight=weight, reduction=reduction,
                                        temperature=kw.get("tau", 1.0), z_loss_weight=kw.get("z", 0.0),
                                        logit_scale=kw.get("scale", 1.0))
    # (without a gradient a weighted call may leave zero-weight tokens out, which splits the vocabulary's sums
    # differently: both are held to the tolerance, not to each other's bits)
    close(same, want, tol["loss"])
    return loss.detach(), grads


DTYPES = [torch.bfloat16, torch.float16, torch.float32]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N,K,V,T", [(1, 8, 1, 1), (1, 64, 1000, 1), (2, 16, 7, 7), (31, 72, 300, 3), (33, 100, 257, 65),
                                     (130, 256, 4097, 9), (257, 128, 2000, 64), (513, 64, 1500, 5), (700, 33, 3000, 2),
                                     (20, 1024, 9000, 130)])
def test_types_and_sizes(dtype, N, K, V, T):
    x = make(N, K, V, T, dtype, seed=N + V)
    check(*x, reduction="sum")
    check(*x, reduction="sum", tau=2.0, z=0.01, scale=0.7)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("reduction", ["none", "sum", "mean"])
@pytest.mark.parametrize("weighted", [False, True])
def test_reductions_weights_and_bias(dtype, bias, reduction, weighted):
    h, W, b, t, ids = make(190, 96, 700, 6, dtype, bias=bias)
    ids[::5] = -1                          # tokens without a teacher
    weight = (2 * torch.rand(190, device=DEV, generator=gen(1))) * (torch.rand(190, device=DEV, generator=gen(2)) > 0.3)
    g = torch.randn(190, device=DEV, generator=gen(3)) if reduction == "none" else torch.tensor(37.0, device=DEV)
    check(h, W, b, t, ids, reduction=reduction, weight=weight if weighted else None, g=g, z=1e-3)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N,V,chunk", [(300, 5000, 256), (600, 5000, 1024), (64, 20000, None), (1100, 9000, 8192)])
def test_chunks_of_the_vocabulary(dtype, N, V, chunk):
    """The teacher's elements of dS in the first, middle and last chunk, on their borders too."""
    h, W, b, t, ids = make(N, 64, V, 8, dtype)
    ids[:, 0], ids[:, 1], ids[:, 2], ids[:, 3] = 0, V - 1, 255, 256
    check(h, W, b, t, ids, reduction="sum", chunk_size=chunk)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N,K,V", [(1, 512, 40000), (32, 256, 9000), (33, 256, 9000), (129, 1024, 3001), (500, 1024, 2500),
                                   (513, 1032, 700)])
@pytest.mark.parametrize("reduction", ["none", "mean"])
def test_kept_scores(dtype, N, K, V, reduction):
    """Few tokens on wide rows: the backward takes the forward's scores, over one chunk and several, with tokens left
    out; a given chunk recomputes them, to the same tolerance."""
    from swvr_amd import _lib
    assert _lib.load().swvr_distill_scores_size(_lib.DTYPE_TAG[dtype], _lib.DTYPE_TAG[dtype], N, K, V, K) > 0
    h, W, b, t, ids = make(N, K, V, 6, dtype, seed=K)
    ids[:, 0], ids[:, 1] = V - 1, 8191 % V
    ids[1::7] = -1
    weight = (torch.rand(N, device=DEV, generator=gen(1)) > 0.3).float()
    weight[0] = 1.0
    g = torch.randn(N, device=DEV, generator=gen(3)) if reduction == "none" else torch.tensor(float(N), device=DEV)
    for chunk in (None, 4096):
        check(h, W, b, t, ids, reduction=reduction, weight=weight, g=g, chunk_size=chunk, tau=1.5, z=1e-3)
    check(h, W, None, t, ids, reduction=reduction, g=g)


@pytest.mark.parametrize("N,K,V", [(1500, 136, 700), (1500, 136, 9001)])
@pytest.mark.parametrize("weighted", [False, True])
def test_fp32_scores_of_many_tokens(N, K, V, weighted):
    """fp32 keeps more of them where no weight may drop tokens; the same gradients either way."""
    from swvr_amd import _lib
    assert _lib.load().swvr_distill_scores_size(_lib.F32, _lib.F32, N, K, V, K) == 1536 * V * 4 > 2 * V * K * 4
    h, W, b, t, ids = make(N, K, V, 5, torch.float32, seed=N)
    ids[::9] = -1
    weight = (torch.rand(N, device=DEV, generator=gen(1)) > 0.5).float() if weighted else None
    check(h, W, b, t, ids, reduction="sum", weight=weight, tau=1.5)
    check(h, W, b, t, ids, reduction="sum", weight=weight, chunk_size=512)


def test_scores_are_kept_only_where_they_are_small():
    from swvr_amd import _lib
    size = lambda *a: _lib.load().swvr_distill_scores_size(*a)
    assert size(_lib.BF16, _lib.BF16, 500, 1024, 32000, 1024) == 512 * 32000 * 4
    assert size(_lib.BF16, _lib.BF16, 512, 512, 32000, 512) == 512 * 32000 * 4
    assert size(_lib.BF16, _lib.BF16, 513, 512, 32000, 512) == 0       # over twice W
    assert size(_lib.BF16, _lib.BF16, 769, 4096, 32000, 4096) == 0     # not the one-pass forward
    assert size(_lib.F32, _lib.F32, 2000, 1024, 32000, 1024) == 2048 * 32000 * 4
    assert size(_lib.F32, _lib.F32, 2000, 1024, 66000, 1024) == 0      # over 512 MB
    assert size(_lib.BF16, _lib.F32, 64, 1024, 32000, 1024) == 0       # W rounded on the way
    assert size(_lib.BF16, _lib.BF16, 64, 1024, 32000, 1 << 24) == 0   # rows too far apart for that forward
    assert size(_lib.F64, _lib.F64, 64, 1024, 32000, 1024) == 0


def test_one_entry_is_cross_entropy():
    h, W, b, _, ids = make(200, 64, 900, 1, torch.float32, absent=0.0)
    loss, (gh, gW, gb) = check(h, W, b, torch.zeros(200, 1, device=DEV), ids)
    xs = [x.detach().double().requires_grad_(True) for x in (h, W, b)]
    want = torch.nn.functional.cross_entropy(xs[0] @ xs[1].t() + xs[2], ids[:, 0])
    for got, w in zip((loss, gh, gW, gb), (want, *torch.autograd.grad(want, xs))):
        assert rel_err(got, w) < 1e-5


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_a_student_that_has_learned(dtype):
    """p = softmax(S) over every id: dS is the difference of two equal terms, rounded once."""
    h, W, b, _, _ = make(40, 64, 50, 1, dtype)
    S = h.double() @ W.double().t() + b.double()
    ids = torch.arange(50, device=DEV).expand(40, 50)
    loss, grads = check(h, W, b, S.float(), ids, reduction="sum")
    assert abs(loss.item()) < 40 * 1e-4
    assert all(x.abs().max().item() < 1e-2 for x in grads)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_ids_that_repeat_in_a_list(dtype):
    h, W, b, t, ids = make(150, 64, 12, 30, dtype)   # 30 entries over 12 ids
    check(h, W, b, t, ids, reduction="sum")
    check(h, W, b, t, torch.full_like(ids, 5), reduction="sum")
    hot = torch.where(torch.rand(150, 30, device=DEV) < 0.5, 3, ids)
    check(h, W, b, t, hot, reduction="sum")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rows_without_a_teacher(dtype):
    h, W, b, t, ids = make(70, 64, 300, 4, dtype)
    t[::3] = -math.inf                    # present ids, no logits
    ids[1::3] = -1
    loss, (gh, _, _) = check(h, W, b, t, ids)
    assert (gh[::3] == 0).all() and (gh[1::3] == 0).all() and (gh[2::3] != 0).any()
    ids[:] = -1                           # nothing to learn from: zero, not 0 / 0
    for reduction in ("mean", "sum"):
        loss, grads = check(h, W, b, t, ids, reduction=reduction)
        assert loss.item() == 0 and all((x == 0).all() for x in grads)
    loss, grads = check(h, W, b, t, make(70, 64, 300, 4, dtype)[4], weight=torch.zeros(70, device=DEV))
    assert loss.item() == 0 and all((x == 0).all() for x in grads)


@pytest.mark.parametrize("N", [70, 900])
def test_dropped_tokens_may_hold_anything(N):
    """Weight zero, or no entries: infinities and NaN there reach nothing."""
    h, W, b, t, ids = make(N, 64, 300, 4, torch.bfloat16)
    weight = torch.ones(N, device=DEV)
    weight[::4] = 0
    want, want_g = check(h, W, b, t, ids, weight=weight)
    t2, ids2 = t.clone(), ids.clone()
    t2[::4], ids2[::4] = math.nan, 10 ** 9
    got, got_g = check(h, W, b, t2, ids2, weight=weight)
    assert torch.equal(got, want) and all(torch.equal(a, c) for a, c in zip(got_g, want_g))
    h2 = h.clone()
    h2[::8], h2[4::8] = math.nan, math.inf
    h2.requires_grad_(True), W.requires_grad_(True), b.requires_grad_(True)
    loss = swvr_amd.softmax_distill(h2, W, t2, ids2, b, weight=weight)
    got_g = torch.autograd.grad(loss, (h2, W, b))
    assert rel_err(loss, want) < 1e-6 and all(rel_err(a, c) < 1e-2 for a, c in zip(got_g, want_g))


def test_ids_beyond_the_vocabulary_show():
    h, W, b, t, ids = make(30, 64, 300, 4, torch.float32, absent=0.0)
    ids[7, 2] = 300
    loss = swvr_amd.softmax_distill(h, W, t, ids, b, reduction="none")
    assert torch.isnan(loss[7]) and torch.isfinite(loss[torch.arange(30, device=DEV) != 7]).all()
    ids[7, 2] = 2 ** 32 + 5               # 5, if it were cut to 32 bits
    assert torch.isnan(swvr_amd.softmax_distill(h, W, t, ids, b))
    t[7, 2] = -math.inf                   # an absent entry's id is not looked at
    check(h, W, b, t, ids, reduction="sum")


def test_masked_student_ids():
    """A bias of -inf masks ids: never probable; a teacher that names one has an infinite divergence there."""
    h, W, b, t, ids = make(60, 64, 200, 5, torch.float32, absent=0.0)
    b[:100] = -math.inf
    ids = ids % 100 + 100
    loss = swvr_amd.softmax_distill(h, W, t, ids, b)
    xs = [x.detach().double().requires_grad_(True) for x in (h, W, b)]
    S = xs[0] @ xs[1].t() + xs[2]
    p = torch.softmax(t.double(), dim=1)
    want = (p * (p.log() - torch.log_softmax(S, dim=1).gather(1, ids))).sum(dim=1).mean()
    assert abs(loss.item() - want.item()) < 1e-5 * abs(want.item())
    h.requires_grad_(True), W.requires_grad_(True)
    gh, gW = torch.autograd.grad(swvr_amd.softmax_distill(h, W, t, ids, b), (h, W))
    wh, wW = torch.autograd.grad(want, xs[:2])
    assert rel_err(gh, wh) < 1e-5 and rel_err(gW, wW) < 1e-5 and (gW[:100] == 0).all()
    ids[3, 0] = 7
    terms = swvr_amd.softmax_distill(h, W, t, ids, b, reduction="none")
    assert terms[3].item() == math.inf and torch.isfinite(terms[:3]).all()


def test_gradient_against_differences():
    h, W, b, t, ids = make(6, 8, 11, 3, torch.float32, absent=0.0)
    kw = dict(temperature=1.5, z_loss_weight=0.05, logit_scale=0.8)
    h.requires_grad_(True), W.requires_grad_(True), b.requires_grad_(True)
    grads = torch.autograd.grad(swvr_amd.softmax_distill(h, W, t, ids, b, **kw), (h, W, b))
    # central differences of the formula in 64 bits, step 1e-5: off by its square and 2^-53 / step
    args = dict(tau=1.5, z=0.05, scale=0.8)
    with torch.no_grad():
        for name, x, got in zip("hWb", (h, W, b), grads):
            flat, num = x.double().reshape(-1), []
            for i in range(flat.numel()):
                vals = []
                for d in (1e-5, -1e-5):
                    y = flat.clone()
                    y[i] += d
                    S = dict(h=h, W=W, b=b)
                    S[name] = y.view(x.shape)
                    vals.append(_loss64(S["h"], S["W"], S["b"], t, ids, **args))
                num.append((vals[0] - vals[1]) / 2e-5)
            assert rel_err(got.reshape(-1), torch.stack(num)) < 1e-5


def _loss64(h, W, b, t, ids, tau, z, scale):
    S = (scale * h.double() @ W.double().t() + b.double()) / tau
    lse = torch.logsumexp(S, dim=1)
    p = torch.softmax(t.double() / tau, dim=1)
    return ((p * (p.log() - S.gather(1, ids) + lse[:, None])).sum(dim=1) + z * lse.square()).mean()


def test_list_types_strides_and_leading_shapes():
    h, W, b, t, ids = make(24, 64, 300, 6, torch.bfloat16)
    want, want_g = check(h, W, b, t, ids)
    wide = torch.full((24, 20), 299, device=DEV)
    wide[:, 4:16:2] = ids
    for i2 in (ids.int(), ids.short(), wide[:, 4:16:2], ids.t().contiguous().t()):
        got, got_g = check(h, W, b, t, i2)
        assert torch.equal(got, want) and all(torch.equal(a, c) for a, c in zip(got_g, want_g))
    for t2 in (t.double(), t.t().contiguous().t(), torch.cat([t, t], dim=1)[:, :6]):
        assert torch.equal(check(h, W, b, t2, ids)[0], want)
    check(h, W, b, t.bfloat16(), ids)
    check(h, W, b, t.half(), ids)
    check(h, W, b, t[:1].expand(24, 6), ids[:1].expand(24, 6))
    lead = swvr_amd.softmax_distill(h.view(2, 3, 4, 64), W, t.view(2, 3, 4, 6), ids.view(2, 3, 4, 6), b,
                                    weight=torch.ones(2, 3, 4, device=DEV), reduction="none")
    flat = swvr_amd.softmax_distill(h, W, t, ids, b, weight=torch.ones(24, device=DEV), reduction="none")
    assert lead.shape == (2, 3, 4) and torch.equal(lead.reshape(-1), flat)
    one = swvr_amd.softmax_distill(h[3], W, t[3], ids[3], b, reduction="none")
    assert one.shape == () and abs(one.item() - flat[3].item()) <= 1e-5 * abs(flat[3].item())


def test_no_tokens():
    h, W, b, t, ids = make(0, 64, 300, 6, torch.bfloat16)
    for reduction in ("mean", "sum", "none"):
        h.requires_grad_(True), W.requires_grad_(True), b.requires_grad_(True)
        loss = swvr_amd.softmax_distill(h, W, t, ids, b, reduction=reduction)
        assert loss.shape == ((0,) if reduction == "none" else ()) and loss.sum().item() == 0
        gh, gW, gb = torch.autograd.grad(loss.sum(), (h, W, b))
        assert gh.shape == (0, 64) and (gW == 0).all() and (gb == 0).all()


@pytest.mark.parametrize("wrt", ["h", "W", "b", "hW", "hb", "Wb"])
def test_frozen_inputs(wrt):
    x = dict(zip(("h", "W", "b", "t", "ids"), make(120, 64, 700, 6, torch.bfloat16)))
    full = dict(zip("hWb", check(*x.values())[1]))
    xs = [x[k].detach().requires_grad_(True) if k in wrt else x[k] for k in "hWb"]
    loss = swvr_amd.softmax_distill(xs[0], xs[1], x["t"], x["ids"], xs[2])
    for k, got in zip(wrt, torch.autograd.grad(loss, [xs["hWb".index(k)] for k in wrt])):
        assert rel_err(got, full[k]) < 1e-2


def test_autocast_with_fp32_parameters():
    h, W, b, t, ids = make(300, 72, 900, 6, torch.float32)
    for cdt in (torch.bfloat16, torch.float16):
        xs = [x.detach().requires_grad_(True) for x in (h, W, b)]
        with torch.autocast("cuda", dtype=cdt):
            loss = swvr_amd.softmax_distill(xs[0], xs[1], t, ids, xs[2], reduction="sum", temperature=1.5)
        grads = torch.autograd.grad(loss, xs)
        want, want_g, tol = formula(h, W, b, t, ids, reduction="sum", tau=1.5, cdt=cdt)
        close(loss.detach(), want, tol["loss"])
        for name, got in zip("hWb", grads):
            assert got.dtype == torch.float32
            close(got, want_g[name], tol[name])


def test_the_same_on_every_run():
    x = make(900, 128, 3000, 16, torch.bfloat16)
    loss, grads = check(*x)
    for _ in range(2):
        again, more = check(*x)
        assert torch.equal(loss, again) and all(torch.equal(a, c) for a, c in zip(grads, more))


def test_another_stream():
    x = make(200, 64, 900, 6, torch.bfloat16)
    loss, grads = check(*x)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other, more = check(*x)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(loss, other) and all(torch.equal(a, c) for a, c in zip(grads, more))


def test_two_streams_at_once():
    """Two calls in flight on two streams, of the same tensors and of others, give what each gives alone."""
    xs = [make(300, K, 4000, 6, torch.bfloat16, seed=K) for K in (64, 1024)]
    want = [check(*x) for x in xs]
    streams = [torch.cuda.Stream() for _ in xs]
    for _ in range(3):
        got = []
        for s in streams:
            s.wait_stream(torch.cuda.current_stream())
        for s, (h, W, b, t, ids) in zip(streams, xs):
            with torch.cuda.stream(s):
                leaves = [x.detach().requires_grad_(True) for x in (h, W, b)]
                loss = swvr_amd.softmax_distill(leaves[0], leaves[1], t, ids, leaves[2])
                got.append((loss.detach(), torch.autograd.grad(loss, leaves)))
        torch.cuda.synchronize()
        for (loss, grads), (l0, g0) in zip(got, want):
            assert torch.equal(loss, l0) and all(torch.equal(a, c) for a, c in zip(grads, g0))


def test_parameters_changed_before_the_backward_are_refused():
    for which in range(3):
        h, W, b, t, ids = make(40, 64, 500, 4, torch.float32)
        xs = [x.requires_grad_(True) for x in (h, W, b)]
        loss = swvr_amd.softmax_distill(h, W, t, ids, b)
        with torch.no_grad():
            xs[which].add_(1)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()


@pytest.mark.parametrize("tau", [1.0, 2.0])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_bias_that_is_a_view(dtype, tau):
    """At temperature 1 a dense fp32 bias is read as it is; others are laid out and scaled first."""
    h, W, b, t, ids = make(60, 64, 500, 4, torch.float32)
    for view in (torch.stack([b, -b], dim=1).to(dtype)[:, 0], torch.cat([b, b]).to(dtype)[499:999], b[:1].to(dtype).expand(500)):
        check(h, W, view, t, ids, tau=tau)


def test_double_backward_is_refused():
    h, W, b, t, ids = make(20, 64, 90, 4, torch.float32)
    h.requires_grad_(True)
    loss = swvr_amd.softmax_distill(h, W, t, ids, b)
    (gh,) = torch.autograd.grad(loss, h, create_graph=True)
    with pytest.raises(RuntimeError):   # there is no graph to go back through
        gh.sum().backward()


def test_log_normalisers_of_a_readout_without_columns():
    """An embedding of width 0: LSE alone, as with columns, and h's and W's gradients through it."""
    for dtype, N in ((torch.bfloat16, 40), (torch.float32, 300), (torch.bfloat16, 900)):
        h, W, b, _, _ = make(N, 64, 700, 1, dtype)
        E = torch.randn(700, 16, device=DEV).to(dtype)
        h.requires_grad_(True), W.requires_grad_(True)
        _, lse0 = swvr_amd.softmax_readout(h, W, E[:, :0], b)
        _, lse = swvr_amd.softmax_readout(h, W, E, b)
        S = h.double() @ W.double().t() + b.double()
        want = torch.logsumexp(S, dim=1)
        assert rel_err(lse0, want) < 1e-6 and rel_err(lse, want) < 1e-6
        g0, g = (torch.autograd.grad(x.sum(), (h, W)) for x in (lse0, lse))
        assert all(rel_err(a, c) < 1e-2 for a, c in zip(g0, g))


def test_compiled_whole():
    h, W, b, t, ids = make(200, 64, 900, 6, torch.bfloat16)
    want, want_g = check(h, W, b, t, ids, chunk_size=8192)
    xs = [x.detach().requires_grad_(True) for x in (h, W, b)]
    loss = torch.compile(lambda a, c, d: swvr_amd.softmax_distill(a, c, t, ids, d), fullgraph=True)(*xs)
    assert torch.equal(loss.detach(), want)
    for got, w in zip(torch.autograd.grad(loss, xs), want_g):
        assert torch.equal(got, w)


@pytest.mark.parametrize("K", [64, 1024])   # scores formed again, and kept
def test_captured_and_replayed(K):
    h, W, b, t, ids = make(300, K, 900, 6, torch.bfloat16)
    for x in (h, W, b):
        x.requires_grad_(True)

    def step():
        loss = swvr_amd.softmax_distill(h, W, t, ids, b, weight=weight)
        return (loss.detach(), *torch.autograd.grad(loss, (h, W, b)))

    weight = torch.ones(300, device=DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for k in range(4):
        with torch.no_grad():
            h.normal_(generator=gen(k))
            t.normal_(generator=gen(10 + k))
            ids.copy_(torch.randint(-1, 900, (300, 6), device=DEV, generator=gen(20 + k)))
            weight.copy_((torch.rand(300, device=DEV, generator=gen(30 + k)) > 0.1 * k).float())
        graph.replay()
        torch.cuda.synchronize()
        for a, c in zip(got, step()):
            assert torch.equal(a, c)


def test_tokens_all_the_way():
    """The three together on a tied table: embed the prompt, train the head on a teacher, draw the next tokens and
    embed those, against the same in 64 bits."""
    V, D, N, T = 700, 64, 40, 8
    g = gen(5)
    E = (0.5 * torch.randn(V, D, device=DEV, generator=g)).requires_grad_(True)
    prompt = torch.randint(-1, V, (N,), device=DEV, generator=g)
    teacher, ids = torch.randn(N, T, device=DEV, generator=g), torch.randint(0, V, (N, T), device=DEV, generator=g)
    h = torch.tanh(swvr_amd.embedding_lookup(prompt, E, scale=2.0))
    loss = swvr_amd.softmax_distill(h, E, teacher, ids, temperature=2.0)
    (gE,) = torch.autograd.grad(loss, E)
    E64 = E.detach().double().requires_grad_(True)
    x64 = torch.where((prompt >= 0)[:, None], 2.0 * E64[prompt.clamp(min=0)], 0.0)
    logq = torch.log_softmax(torch.tanh(x64) @ E64.t() / 2.0, dim=1)
    p = torch.softmax(teacher.double() / 2.0, dim=1)
    want = (p * (p.log() - logq.gather(1, ids))).sum(dim=1).mean()
    assert rel_err(loss, want) < 1e-5
    assert rel_err(gE, torch.autograd.grad(want, E64)[0]) < 1e-5
    with torch.no_grad():
        logits = h @ E.t()
        u = torch.rand(N, device=DEV, generator=g)
        token, logprob = swvr_amd.sample_tokens(logits, u, top_k=10)
        top = logits.topk(10, dim=1).indices
        assert ((token[:, None] == top).any(dim=1)).all()
        kept = torch.log_softmax(logits.double().gather(1, top), dim=1)
        assert torch.allclose(logprob.double(), kept[token[:, None] == top], atol=1e-6)
        nxt = swvr_amd.embedding_lookup(token, E, scale=2.0)
        assert torch.equal(nxt, 2.0 * E[token])
