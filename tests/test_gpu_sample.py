"""sample_tokens on the GPU against the definition in 64 bits, row by row: filters alone and together, ties, masks of
-inf, NaN, infinities and the types' lowest values, rows with nothing to draw, lengths from one, views off every
alignment, settings per row, graphs and compilation.

Tokens must be equal.  logprob: fp32 of a 64-bit value whose sum of weights is rounded to multiples of 2^-44 of the
largest: half a step of fp32, relative, and 1e-7 for the sum."""
import math

import pytest
import torch

import swvr_amd

pytestmark = pytest.mark.gpu
DEV = "cuda"


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def want_row(x, u, tau, k, p, min_p):
    """(token, logprob) of one row by the definition."""
    x = x.double().cpu()
    x = torch.where(x.isnan(), -math.inf, x)
    if x.max() == -math.inf:
        return -1, -math.inf
    order = torch.argsort(-x, stable=True)
    m = x[order[0]]
    if not tau > 0:
        return int(order[0]), 0.0
    w = torch.where(x[order] == m, 1.0, torch.exp((x[order] - m) / tau))
    w = torch.where(x[order] == -math.inf, 0.0, w).nan_to_num(0.0)
    n = w.numel()
    if 0 < k < n:
        w = w[:k]
    if p < 1:
        before = w.cumsum(0) - w
        w = w[:max(1, int((before < p * w.sum()).sum()))]
    if min_p > 0:
        w = w[:max(1, int((w >= min_p).sum()))]
    kept, back = order[:w.numel()].sort()
    w = w[back]
    run = w.cumsum(0)
    target = min(u, 1 - 2.0 ** -53) * run[-1]
    j = int((run <= target).sum())
    return int(kept[j]), float(torch.log(w[j] / run[-1]))


def check(logits, u, **kw):
    token, logprob = swvr_amd.sample_tokens(logits, u, **kw)
    assert token.dtype == torch.int64 and logprob.dtype == torch.float32 and token.shape == logprob.shape == u.shape
    flat, uu = logits.reshape(-1, logits.shape[-1]), u.reshape(-1)

    def of(name, i, default):
        x = kw.get(name)
        return default if x is None else x.reshape(-1)[i].item() if isinstance(x, torch.Tensor) else x

    for i in range(flat.shape[0]):
        t, lp = want_row(flat[i], uu[i].item(), of("temperature", i, 1.0), of("top_k", i, 0), of("top_p", i, 1.0),
                         of("min_p", i, 0.0))
        got, got_lp = token.reshape(-1)[i].item(), logprob.reshape(-1)[i].item()
        assert got == t, (i, got, t)
        assert got_lp == lp or abs(got_lp - lp) <= 2.0 ** -24 * abs(lp) + 1e-7, (i, got_lp, lp)
    return token, logprob


FILTERS = [dict(), dict(temperature=0.0), dict(temperature=0.3), dict(temperature=2.5), dict(top_k=1), dict(top_k=7),
           dict(top_k=300), dict(top_k=10 ** 9), dict(top_p=0.0), dict(top_p=0.4), dict(top_p=0.97), dict(min_p=0.02),
           dict(min_p=1.0), dict(top_k=40, top_p=0.9), dict(top_k=40, top_p=0.9, min_p=0.1, temperature=0.8),
           dict(top_p=0.99, min_p=0.001, temperature=1.5), dict(top_k=2000, top_p=0.8)]


@pytest.mark.parametrize("kw", FILTERS, ids=str)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("R,V", [(3, 1), (5, 2), (4, 63), (3, 1000), (2, 4097), (2, 50257)])
def test_filters_types_and_lengths(kw, dtype, R, V):
    x = (3 * torch.randn(R, V, device=DEV, generator=gen(V + R))).to(dtype)
    check(x, torch.rand(R, device=DEV, generator=gen(R)), **kw)


@pytest.mark.parametrize("kw", [dict(), dict(top_k=50, top_p=0.9), dict(top_p=0.95), dict(top_k=5000, top_p=0.5),
                                dict(min_p=0.05), dict(top_k=1)], ids=str)
@pytest.mark.parametrize("spread", [0.0, 0.01, 1.0, 6.0, 60.0])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_large_vocabulary_flat_to_peaked(kw, spread, dtype):
    """From all logits equal (every token a tie) to one token with all of the weight."""
    x = (spread * torch.randn(3, 151936, device=DEV, generator=gen(5))).to(dtype)
    check(x, torch.tensor([0.1, 0.617, 0.98], device=DEV), **kw)


@pytest.mark.parametrize("kw", [dict(top_k=3), dict(top_k=500), dict(top_k=5001), dict(top_p=0.3), dict(top_p=0.9),
                                dict(top_k=6000, top_p=0.7), dict()], ids=str)
def test_ties_at_every_cut(kw):
    """Few distinct logits: the cuts fall inside runs of equal ones, which go by index."""
    x = torch.randint(0, 3, (6, 20000), device=DEV, generator=gen(6)).float()
    check(x, torch.rand(6, device=DEV, generator=gen(7)), **kw)
    check(x.bfloat16() * -1000, torch.rand(6, device=DEV, generator=gen(8)), **kw)


@pytest.mark.parametrize("kw", [dict(), dict(top_k=50), dict(top_k=50, top_p=0.9), dict(top_k=150, top_p=0.9), dict(top_p=0.6),
                                dict(top_k=4000, top_p=0.99, min_p=0.2), dict(top_p=0.95, min_p=0.3)], ids=str)
@pytest.mark.parametrize("spread", [0.0, 0.01, 1.0, 60.0])
@pytest.mark.parametrize("V,off", [(257, 0), (2049, 1), (4095, 2), (4096, 3), (4096, 7)])
def test_short_rows_flat_to_peaked(kw, spread, V, off):
    """Rows that fit one workgroup's list, up to a full one, beginning anywhere between two borders of loads."""
    g = gen(V + off)
    x = (spread * torch.randn(4, V + 9, device=DEV, generator=g)).bfloat16()
    x[1] = x[1].sign()
    check(x[:, off:off + V], torch.rand(4, device=DEV, generator=g), **kw)


@pytest.mark.parametrize("kw", [dict(), dict(top_k=4), dict(top_p=0.8), dict(min_p=0.3), dict(temperature=0.0)], ids=str)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("V", [3001, 20011])   # a row in one launch, and in several
def test_masked_infinite_and_nan_logits(kw, dtype, V):
    x = torch.randn(10, V, device=DEV, generator=gen(9)).to(dtype)
    x[0] = -math.inf                                # nothing to draw
    x[1] = math.nan                                 # nothing to draw
    x[2] = -math.inf
    x[2, 1234] = -5                                 # one token left
    x[3, ::2] = -math.inf
    x[4, 7::3] = math.nan
    x[5, 100], x[5, 2000] = math.inf, math.inf      # two infinite ones share the weight
    x[6] = torch.finfo(dtype).min                   # masked with the lowest value throughout
    x[7, :] = torch.finfo(dtype).min
    x[7, [5, 900]] = 1.0
    x[8, 0], x[8, 1] = torch.finfo(dtype).max, torch.finfo(dtype).min
    x[9, ::2], x[9, 1::2] = 0.0, -0.0               # zeros of both signs tie
    for seed in range(3):
        token, logprob = check(x, torch.rand(10, device=DEV, generator=gen(seed)), **kw)
        assert token[:2].tolist() == [-1, -1] and logprob[0].item() == -math.inf


def test_ends_of_u():
    x = torch.randn(5, 777, device=DEV, generator=gen(10))
    x[:, 0] = x[:, -1] = -math.inf
    u = torch.tensor([0.0, 1 - 2.0 ** -24, 1.0, 0.5, 2.0 ** -149], device=DEV)
    check(x, u)
    check(x, u, top_k=20)
    check(x, u.double())
    token, _ = swvr_amd.sample_tokens(x, torch.tensor([0.0, -1.0, math.nan, math.inf, 7.0], device=DEV))
    assert token.tolist() == [1, 1, 1, 775, 775]


def test_settings_of_each_row():
    R, V = 24, 5000
    g = gen(11)
    pick = lambda values: torch.tensor(values, device=DEV)[torch.randint(0, len(values), (R,), device=DEV, generator=g)]
    x = 2 * torch.randn(R, V, device=DEV, generator=g)
    u = torch.rand(R, device=DEV, generator=g)
    kw = dict(temperature=pick([0.0, 0.5, 1.0, -1.0, math.nan]), top_k=pick([0, 1, 30, 3000, -2, 10 ** 6]),
              top_p=pick([1.0, 0.5, 0.95]), min_p=pick([0.0, 0.05]))
    want, _ = check(x, u, **kw)
    for dtype in (torch.int32, torch.int16):
        token, _ = swvr_amd.sample_tokens(x, u, **{**kw, "top_k": kw["top_k"].clamp(-2, 5000).to(dtype)})
        assert torch.equal(token, want)
    huge = torch.where(kw["top_k"] == 10 ** 6, 2 ** 32 + 1, kw["top_k"])   # 1, if it were cut to 32 bits
    assert torch.equal(swvr_amd.sample_tokens(x, u, **{**kw, "top_k": huge})[0], want)
    over = swvr_amd.sample_tokens(x, u, min_p=torch.full_like(u, 7.0))[0]
    assert torch.equal(over, x.argmax(dim=1))
    # a row alone gives what it gives in the batch, whatever the layout
    for i in range(0, R, 5):
        one, _ = swvr_amd.sample_tokens(x[i], u[i], **{k: v[i] for k, v in kw.items()})
        assert one.shape == () and one == want[i]
    lead = {k: v.view(2, 12) for k, v in kw.items()}
    token, _ = check(x.view(2, 12, V), u.view(2, 12), **lead)
    assert torch.equal(token.view(-1), want)


@pytest.mark.parametrize("R,V", [(2 ** 21 + 7, 3), (2100, 4100)])   # more rows than one launch takes
def test_many_rows(R, V):
    g = gen(21)
    x = 2 * torch.randn(R, V, device=DEV, generator=g).bfloat16()
    u = torch.rand(R, device=DEV, generator=g)
    kw = dict(temperature=torch.rand(R, device=DEV, generator=g), top_p=torch.rand(R, device=DEV, generator=g),
              min_p=0.1 * torch.rand(R, device=DEV, generator=g), top_k=torch.randint(1, V, (R,), device=DEV, generator=g))
    token, logprob = swvr_amd.sample_tokens(x, u, **kw)
    assert int(token.min()) >= 0 and int(token.max()) < V and bool((logprob <= 0).all())
    for rows in (slice(0, 5), slice(R // 2, R // 2 + 5), slice(R - 9, R)):
        t, lp = check(x[rows], u[rows], **{k: v[rows] for k, v in kw.items()})
        assert torch.equal(t, token[rows]) and torch.equal(lp, logprob[rows])


@pytest.mark.parametrize("kw", [dict(), dict(top_k=40, top_p=0.9), dict(top_p=0.7, min_p=0.01), dict(temperature=0.0)], ids=str)
@pytest.mark.parametrize("V", [2 ** 21 - 8, 2 ** 21 + 5])   # the longest rows of the launches for many workgroups; longer
def test_the_longest_rows(kw, V):
    x = 3 * torch.randn(2, V, device=DEV, generator=gen(24))
    check(x, torch.rand(2, device=DEV, generator=gen(25)), **kw)


@pytest.mark.parametrize("V", [1000, 9000])
def test_many_draws_from_one_row(V):
    x = torch.randn(V, device=DEV, generator=gen(22)).expand(7, V)
    check(x, torch.rand(7, device=DEV, generator=gen(23)), top_p=0.9)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_views_off_every_alignment(dtype):
    big = (3 * torch.randn(6, 9000, device=DEV, generator=gen(12))).to(dtype)
    u = torch.rand(6, device=DEV, generator=gen(13))
    for lo in range(9):
        for n in (1, 5, 4093, 4097, 8990):
            check(big[:, lo:lo + n], u, top_p=0.9)
    check(big[:, ::3], u, top_k=9)
    check(big[::2], u[::2])
    check(big[:1].expand(6, 9000), u, top_p=0.7)
    for kw in (dict(), dict(top_k=30), dict(top_p=0.5), dict(min_p=0.01)):
        for lo in (1, 3, 8):
            check(big[:, lo:lo + 8200], u, **kw)
    check(torch.randn(300, 6, device=DEV, generator=gen(14)).to(dtype).t(), u)


def test_frequencies_follow_the_kept_distribution():
    """20000 draws from one row: every kept token's count within 5 standard deviations, none outside."""
    x = torch.tensor([2.0, -1.0, 0.5, 1.0, -math.inf, 0.5, 3.0], device=DEV)
    n = 20000
    token, _ = swvr_amd.sample_tokens(x.expand(n, 7), torch.rand(n, device=DEV, generator=gen(15)), top_k=5,
                                      temperature=1.3)
    p = torch.softmax(torch.where(x >= 0.5, x, -math.inf).double() / 1.3, 0)
    count = torch.bincount(token, minlength=7).double()
    assert (count[p == 0] == 0).all()
    assert ((count - n * p).abs() <= 5 * (n * p * (1 - p)).sqrt()).all()


def test_no_rows_and_no_gradient():
    token, logprob = swvr_amd.sample_tokens(torch.zeros(0, 9, device=DEV), torch.zeros(0, device=DEV))
    assert token.shape == logprob.shape == (0,)
    x = torch.randn(2, 9, device=DEV, requires_grad=True)
    token, logprob = swvr_amd.sample_tokens(x, torch.rand(2, device=DEV))
    assert not logprob.requires_grad


def test_captured_and_replayed_with_another_stream_beside_it():
    x = torch.randn(8, 30000, device=DEV, generator=gen(16))
    u = torch.rand(8, device=DEV, generator=gen(17))
    settings = [dict(), dict(top_k=50), dict(top_p=0.9), dict(top_k=9000, min_p=0.01)]
    graphs = []
    for kw in settings:  # two graphs alive at once do not share memory that matters
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            swvr_amd.sample_tokens(x, u, **kw)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = swvr_amd.sample_tokens(x, u, **kw)
        graphs.append((graph, out, kw))
    for k in range(3):
        x.normal_(generator=gen(20 + k))
        u.uniform_(generator=gen(30 + k))
        torch.cuda.synchronize()
        for graph, _, _ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for _, (token, logprob), kw in graphs:
            t, lp = check(x, u, **kw)
            assert torch.equal(token, t) and torch.equal(logprob, lp)


def test_compiled_whole():
    x, u = torch.randn(4, 500, device=DEV, generator=gen(18)), torch.rand(4, device=DEV, generator=gen(19))
    want = swvr_amd.sample_tokens(x, u, top_k=40, top_p=0.9)
    got = torch.compile(lambda a, b: swvr_amd.sample_tokens(a, b, top_k=40, top_p=0.9), fullgraph=True)(x, u)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
