"""select_beams and reorder_beams on the GPU against their definitions in 64 bits: sizes from one, ties, masks,
infinities and NaN, finished beams, lengths, rows off every alignment, long rows and wide searches, states of every
type, layout and width, graphs and compilation, and a search that runs them together.

Tokens and parents are equal.  A score is an fp64 sum: exponentials off by 1.1e-12 of themselves, so the lse by that
and roundings of 2^-53 of its size, 2e-12 with them, and 2^-50 of the score; in fp32 half a step of it besides."""
import math

import pytest
import torch

import swvr_amd
from swvr_amd import int8

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = [torch.bfloat16, torch.float16, torch.float32]


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def want_group(x, scores, k, finished, end_id, lengths, alpha):
    """Of one sequence: [(token, parent, score)], k of them."""
    x, found = x.double().cpu(), []
    x = torch.where(x.isnan(), -math.inf, x)
    for w in range(x.shape[0]):
        s = float(scores[w])
        if not math.isfinite(s):
            continue
        n = int(lengths[w]) if lengths is not None else 0
        if finished is not None and bool(finished[w]):
            found.append((-s / max(n, 1) ** alpha, w, 0, end_id, s))
            continue
        m = float(x[w].max())
        if not math.isfinite(m):
            continue
        rest = float((x[w] - m).exp().sum().log())   # (of lse = m + rest, which a large m would swallow)
        by = float(max(n + 1, 1)) ** alpha
        order = torch.argsort(-x[w], stable=True)[:k]
        for i, (v, l) in enumerate(zip(order.tolist(), x[w][order].tolist())):
            if l > -math.inf:
                found.append((-((s + ((l - m) - rest)) / by), w, i, v, s + ((l - m) - rest)))
    found.sort()
    found = [(f[3], f[1], f[4]) for f in found[:k]]
    return found + [(-1, -1, -math.inf)] * (k - len(found))


def check(logits, scores, k=None, **kw):
    out = swvr_amd.select_beams(logits, scores, k, **kw)
    W, V = logits.shape[-2:]
    k = k or W
    shape = (*logits.shape[:-2], k)
    assert [x.shape for x in out] == [shape] * 3 and out[0].dtype == out[1].dtype == torch.int64
    assert out[2].dtype == (torch.float64 if scores.dtype == torch.float64 else torch.float32)
    token, parent, score = (x.reshape(-1, k).cpu() for x in out)
    flat, sc = logits.reshape(-1, W, V), scores.reshape(-1, W).cpu().double()

    def of(name, b):
        x = kw.get(name)
        return None if x is None else x.reshape(-1, W)[b].cpu()

    for b in range(flat.shape[0]):
        want = want_group(flat[b], sc[b], k, of("finished", b), kw.get("end_id"), of("lengths", b), kw.get("length_penalty", 0.0))
        assert token[b].tolist() == [f[0] for f in want], b
        assert parent[b].tolist() == [f[1] for f in want], b
        for got, (_, _, s) in zip(score[b].tolist(), want):
            if s == -math.inf:
                assert got == s
                continue
            room = 2e-12 + 2.0 ** -50 * abs(s) + (2.0 ** -24 * abs(s) if out[2].dtype == torch.float32 else 0)
            assert abs(got - s) <= room, (got, s)
    return out


def make(B, W, V, dtype, seed=0, spread=3.0, masked=0.02):
    g = gen(seed + V)
    x = torch.randn(B, W, V, device=DEV, generator=g) * spread
    if masked:
        x[..., torch.rand(V, device=DEV, generator=g) < masked] = -math.inf
    return x.to(dtype), -5 - torch.rand(B, W, device=DEV, generator=g).cumsum(1)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,W,V,k", [(1, 1, 1, 1), (2, 3, 1, 4), (1, 2, 3, 8), (1, 4, 7, 8), (2, 4, 8, 4), (2, 4, 9, 40),
                                     (3, 2, 63, 5), (2, 4, 64, 4), (2, 4, 65, 8), (1, 8, 511, 16), (1, 8, 2047, 16), (1, 8, 2048, 16),
                                     (2, 5, 2049, 10), (3, 4, 8193, 4), (1, 4, 50021, 8), (2, 1, 151936, 1), (1, 3, 65537, 256),
                                     (2, 70, 300, 64), (1, 256, 40, 256), (7, 16, 1000, 32)])
def test_sizes(B, W, V, k, dtype):
    x, s = make(B, W, V, dtype)
    check(x, s, k)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,W,V,k", [(2, 17, 2, 5), (1, 20, 7, 3), (1, 17, 8, 64), (1, 33, 9, 33), (2, 2, 127, 33), (1, 17, 130, 1),
                                     (1, 5, 3001, 250), (2, 64, 2050, 64), (1, 65, 700, 64), (1, 100, 515, 100), (1, 256, 300, 256),
                                     (2, 255, 129, 17), (1, 2, 32000, 256), (1, 256, 64, 1)])
def test_many_beams_and_candidates(B, W, V, k, dtype):
    x, s = make(B, W, V, dtype, seed=7)
    check(x, s, k)
    s[:, 1::3] = -math.inf
    check(x, s - 20 * torch.arange(W, device=DEV), k)     # (the first beams have most)


def test_equal_ranks_of_many_beams():
    x = torch.randn(1, 1, 300, device=DEV, generator=gen(8)).expand(1, 200, 300)
    s = torch.full((1, 200), -1.5, device=DEV)
    _, parent, _ = check(x, s, 256)
    assert parent[0, :200].tolist() == list(range(200))
    check(torch.zeros(1, 40, 9000, device=DEV), s[:, :40], 256)


@pytest.mark.parametrize("V,k", [(262144, 5), (262145, 6), (300001, 256), (2 ** 21, 4)])
def test_long_rows(V, k):
    x, s = make(1, 2, V, torch.float16)
    check(x, s, k)


def test_the_first_step():
    """All beams alike, and only the first counts."""
    x = torch.randn(3, 1, 5001, device=DEV, generator=gen(1)).expand(3, 4, 5001)
    s = torch.full((3, 4), -math.inf, device=DEV)
    s[:, 0] = 0
    token, parent, _ = check(x, s)
    assert (parent == 0).all() and all(len(set(t.tolist())) == 4 for t in token)


@pytest.mark.parametrize("V", [64, 2049, 5001, 30011])
def test_equal_beams_go_by_number(V):
    """Rows of odd lengths begin at other addresses: their sums are the same all the same."""
    x = torch.randn(2, 1, V, device=DEV, generator=gen(2)).expand(2, 5, V).contiguous()
    s = torch.full((2, 5), -3.25, device=DEV)
    _, parent, score = check(x, s, 10)
    assert parent.tolist() == [[0, 1, 2, 3, 4] * 2] * 2
    assert all(len(set(r[:5])) == 1 for r in score.tolist())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V,k", [(40, 9), (3000, 20), (40000, 256), (300000, 7)])
def test_equal_logits_go_by_index(V, k, dtype):
    s = torch.tensor([[-1.0, -2.0]], device=DEV)
    for x in (torch.zeros(1, 2, V, device=DEV), torch.randint(0, 3, (1, 2, V), device=DEV, generator=gen(3)).float(),
              torch.where(torch.rand(1, 2, V, device=DEV, generator=gen(4)) < 0.5, 0.0, -0.0)):
        check(x.to(dtype), s, k)


@pytest.mark.parametrize("k", [1, 16, 256])
def test_logits_in_order(k):
    up = torch.arange(100000, device=DEV).float() * 1e-4
    # all alike but the first of every 64: the best logits lie with few threads, more than a list holds
    few = torch.where(torch.arange(100000, device=DEV) % 64 == 0, 0.0, 5.0)
    steep = torch.linspace(0, -200, 100000, device=DEV)
    far = torch.where(torch.arange(100000, device=DEV) % 2048 < 128, 9.0, 0.0)     # 49 groups of large equal ones
    for x in (up, up.flip(0), few, 5 - few, steep, far):
        check(torch.stack([x, x])[None], torch.tensor([[-4.0, -4.5]], device=DEV), k)


def test_masks_infinities_and_nan():
    x, _ = make(9, 3, 700, torch.float32, seed=5)
    s = torch.full((9, 3), -7.0, device=DEV)
    x[0, 0] = -math.inf                       # a beam with nothing
    x[1] = -math.inf                          # a sequence with nothing
    x[2, 1, 5], x[2, 2, ::2] = math.nan, math.nan
    x[3, 0, 9] = math.inf
    s[4, 0], s[5, 1], s[6, 2] = -math.inf, math.inf, math.nan
    x[7] = torch.finfo(torch.float32).min     # the type's lowest value in a mask
    x[7, 1, 3] = 2.0
    x[8, :, 2:] = -math.inf                   # two candidates a beam
    out = check(x, s, 8)
    assert (out[0][1] == -1).all() and (out[1][1] == -1).all() and (out[2][1] == -math.inf).all()
    check(torch.full((2, 2, 100), math.nan, device=DEV), torch.zeros(2, 2, device=DEV))
    for dtype in (torch.bfloat16, torch.float16):
        y = torch.full((1, 2, 900), torch.finfo(dtype).min, dtype=dtype, device=DEV)
        y[0, 1, 77] = torch.finfo(dtype).max
        check(y, torch.zeros(1, 2, device=DEV), 5)


def test_masks_infinities_and_nan_of_many_candidates():
    x, s = make(6, 20, 3000, torch.float32, seed=11)
    x[0, :, 30:] = -math.inf                  # fewer candidates than are looked for
    x[0, 3:] = -math.inf
    x[1, 0], x[1, 1, ::2], x[1, 2, 77] = math.nan, math.nan, math.inf
    x[2, :, 100:] = torch.finfo(torch.float32).min
    x[3] = -math.inf
    x[3, 19, 2999] = 0.0                      # one in all
    s[4, 1:], s[5, ::2] = -math.inf, math.nan
    out = check(x, s, 100)
    assert (out[0][3] >= 0).sum() == 1 and (out[0][0] >= 0).sum() == 90
    check(x[:, :2], s[:, :2], 40, finished=torch.arange(12, device=DEV).view(6, 2) % 3 == 0, end_id=7)


@pytest.mark.parametrize("k", [3, 100])
def test_equal_logits_of_the_longest_rows(k):
    x = torch.randint(0, 2, (1, 2, 2 ** 21), device=DEV, generator=gen(12)).to(torch.bfloat16)
    x[0, 1] = 0
    check(x, torch.tensor([[-1.0, -2.0]], device=DEV), k)


@pytest.mark.parametrize("far", [-3e38, -4194304.0, -4194303.0, -70000.0, -100.0, 100.0, 70000.0, 4194000.0, 4194304.0, 1e7, 2e38])
def test_logits_far_from_zero(far):
    """Sums do not lose what a large maximum would swallow: differences alone count."""
    x = torch.randn(1, 3, 5000, device=DEV, generator=gen(9)) * 5 + far
    x[0, 1, 3000:] -= 600          # pieces that count for little
    x[0, 2, 2500:4800] = torch.finfo(torch.float32).min
    check(x, torch.tensor([[-3.0, -3.25, -2.0]], device=DEV), 8)


@pytest.mark.parametrize("alpha", [0.0, 0.6, 1.0, 16.0])
def test_finished_beams_and_lengths(alpha):
    x, s = make(6, 4, 3001, torch.bfloat16, seed=6)
    finished = torch.rand(6, 4, device=DEV, generator=gen(7)) < 0.5
    finished[0], finished[1] = True, False
    lengths = torch.randint(0, 40, (6, 4), device=DEV, generator=gen(8))
    check(x, s * 4, 8, finished=finished, end_id=2, lengths=lengths, length_penalty=alpha)
    check(x, s * 4, 8, finished=finished, end_id=3000, lengths=lengths.int(), length_penalty=alpha)
    check(x, s * 4, 3, lengths=lengths.t().contiguous().t(), length_penalty=alpha)
    check(x, s * 4, 6, finished=finished.t().contiguous().t(), end_id=0)
    check(x, -s, 6, lengths=lengths - 20, length_penalty=alpha)       # sums above 0; lengths below 1 count as 1


def test_scores_in_64_bits_and_of_any_size():
    x, s = make(3, 4, 2001, torch.float32, seed=9)
    check(x, s.double() - 1e5 + 1e-7, 8)
    for size in (1e6, 1e9, 3e38):       # (a score so low that fp64 sums with it are equal: the logits decide)
        t = s.clone()
        t[:, 1:] = -size
        token, parent, _ = swvr_amd.select_beams(x, t, 4)
        assert torch.equal(parent, torch.zeros_like(parent))
        assert torch.equal(token, x[:, 0].sort(dim=-1, descending=True, stable=True)[1][:, :4])
    got = swvr_amd.select_beams(x, s.to(torch.bfloat16), 4)
    want = check(x, s.to(torch.bfloat16).float(), 4)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_equal_sums_of_one_beam_go_by_logit():
    """Scores so large that sums with different logits are the same number."""
    x = torch.tensor([[[1.0, 3.0, 2.0, 3.0], [9.0, 8.0, 9.5, 7.0]]], device=DEV)
    token, parent, _ = swvr_amd.select_beams(x, torch.full((1, 2), -1e30, device=DEV), 6)
    assert parent.tolist() == [[0, 0, 0, 0, 1, 1]] and token.tolist() == [[1, 3, 2, 0, 2, 0]]


@pytest.mark.parametrize("dtype", TYPES)
def test_layouts(dtype):
    x, s = make(4, 3, 1001, dtype, seed=10)
    wide = torch.zeros(4, 3, 1012, dtype=dtype, device=DEV)
    for o in range(5):
        wide[..., o:o + 1001] = x
        check(wide[..., o:o + 1001], s, 4)
    check(x.transpose(0, 1).contiguous().transpose(0, 1), s.t().contiguous().t(), 4)
    check(x.transpose(1, 2).contiguous().transpose(1, 2), s, 4)
    check(x[0], s[0], 4)
    check(x.reshape(2, 2, 3, 1001), s.reshape(2, 2, 3), 4)
    check(x[:0], s[:0], 4)
    check(x[:1, :1].expand(2, 3, 1001), s[:2], 4)


def test_many_sequences_of_few_tokens():
    x, s = make(30000, 2, 33, torch.float16, seed=11, masked=0)
    token, parent, score = swvr_amd.select_beams(x, s, 2)
    sums = (s.double()[:, :, None] + torch.log_softmax(x.double(), dim=2)).flatten(1)
    best, at = sums.sort(dim=1, descending=True, stable=True)
    clear = (best[:, 0] - best[:, 1] > 1e-9) & (best[:, 1] - best[:, 2] > 1e-9)
    assert clear.float().mean() > 0.5
    assert torch.equal((parent * 33 + token)[clear], at[clear, :2])
    for part in (slice(0, 10), slice(29000, 30000)):
        assert torch.equal(swvr_amd.select_beams(x[part], s[part], 2)[2], score[part])


def test_the_same_in_any_batch_and_on_every_run():
    x, s = make(5, 4, 40001, torch.float32, seed=12)
    whole = swvr_amd.select_beams(x, s.double(), 8)
    for _ in range(3):
        again = swvr_amd.select_beams(x, s.double(), 8)
        assert all(torch.equal(a, b) for a, b in zip(whole, again))
    for b in range(5):
        one = swvr_amd.select_beams(x[b:b + 1].clone(), s[b:b + 1].double(), 8)
        assert all(torch.equal(a[b:b + 1], c) for a, c in zip(whole, one))


def test_selection_captured_and_replayed():
    x, s = make(3, 4, 20011, torch.bfloat16, seed=13)
    graphs = []
    for k in (4, 9):     # two graphs alive at once do not share memory that matters
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            swvr_amd.select_beams(x, s, k)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = swvr_amd.select_beams(x, s, k)
        graphs.append((graph, out, k))
    for i in range(3):
        x.copy_(torch.randn(x.shape, device=DEV, generator=gen(40 + i)))
        torch.cuda.synchronize()
        for graph, _, _ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for _, out, k in graphs:
            assert all(torch.equal(a, b) for a, b in zip(out, check(x, s, k)))


def test_calls_on_streams_at_once():
    x, s = make(4, 4, 30011, torch.float32, seed=14)
    want = swvr_amd.select_beams(x, s, 4)
    torch.cuda.synchronize()
    outs = []
    for st in [torch.cuda.Stream() for _ in range(4)]:
        with torch.cuda.stream(st):
            outs.append(swvr_amd.select_beams(x, s, 4))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for o in outs for a, b in zip(o, want))


def test_selection_as_traced_and_compiled():
    x, s = make(2, 3, 501, torch.bfloat16, seed=15)
    f, n = torch.rand(2, 3, device=DEV) < 0.5, torch.randint(1, 9, (2, 3), device=DEV)
    for y in (x, x.transpose(0, 1).contiguous().transpose(0, 1)):
        for t in (s, s.double(), s.bfloat16()):
            torch.library.opcheck(torch.ops.swvr.select_beams.default, (y, t, 4, f, 2, n, 0.6), test_utils=("test_schema", "test_faketensor"))
    want = swvr_amd.select_beams(x, s, 4, finished=f, end_id=1, lengths=n, length_penalty=1.0)
    torch._dynamo.reset()
    got = torch.compile(lambda a, b: swvr_amd.select_beams(a * 1, b * 1, 4, finished=f, end_id=1, lengths=n, length_penalty=1.0),
                        fullgraph=True)(x, s)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


# ---------------------------------------------------------------- states
def reordered(x, parents):
    """By the definition, on the CPU."""
    if x.dtype == torch.float8_e4m3fn:      # (as its bytes)
        return reordered(x.view(torch.uint8), parents).view(x.dtype)
    nb = parents.dim() - 1
    x, p = x.detach().cpu(), parents.cpu().long()
    W = x.shape[nb]
    there = (p >= 0) & (p < W)
    flat = x.reshape(math.prod(x.shape[:nb]), W, *x.shape[nb + 1:])
    q = torch.where(there, p, 0).reshape(flat.shape[0], p.shape[-1])
    out = torch.stack([flat[b][q[b]] for b in range(flat.shape[0])]) if flat.shape[0] else flat.new_empty(0, p.shape[-1], *x.shape[nb + 1:])
    out[~there.reshape(out.shape[:2])] = 0
    return out.reshape(*x.shape[:nb], p.shape[-1], *x.shape[nb + 1:])


def same(a, b):
    a, b = a.cpu().contiguous(), b.contiguous()
    return a.shape == b.shape and a.dtype == b.dtype and torch.equal(a.view(torch.uint8) if a.dim() else a, b.view(torch.uint8) if b.dim() else b)


def check_states(xs, parents):
    want = [reordered(x, parents) for x in xs]
    got = swvr_amd.reorder_beams(xs, parents)
    assert isinstance(got, list) and all(same(a, b) for a, b in zip(got, want))
    k, W = parents.shape[-1], xs[0].shape[parents.dim() - 1]
    if k == W and W <= 64:
        assert swvr_amd.reorder_beams(xs, parents, inplace=True) is xs
        assert all(same(a, b) for a, b in zip(xs, want))


def state(shape, dtype, seed=0):
    n = torch.empty(shape, dtype=dtype).numel() * torch.empty((), dtype=dtype).element_size()
    raw = torch.randint(0, 2 if dtype == torch.bool else 256, (n,), device=DEV, generator=gen(seed + n), dtype=torch.uint8)
    return raw.view(dtype).reshape(shape)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32, torch.int64, torch.uint8, torch.bool, torch.float8_e4m3fn,
                                   torch.complex64, torch.complex128, torch.float16])
def test_states_of_any_type(dtype):
    p = torch.randint(-1, 4, (3, 4), device=DEV, generator=gen(50))
    check_states([state((3, 4, 5, 7), dtype), state((3, 4), dtype), state((3, 4, 2, 3, 8), dtype)], p)


@pytest.mark.parametrize("W,k", [(1, 1), (1, 5), (2, 2), (3, 3), (4, 4), (5, 5), (8, 8), (9, 9), (16, 16), (17, 17), (32, 32),
                                 (33, 33), (64, 64), (65, 65), (256, 256), (4, 8), (8, 4), (10, 100), (256, 1), (1, 256)])
def test_numbers_of_beams(W, k):
    p = torch.randint(0, W, (3, k), device=DEV, generator=gen(W + k))
    check_states([state((3, W, 4, 24), torch.bfloat16), state((3, W, 5), torch.uint8)], p)


@pytest.mark.parametrize("n", [1, 2, 3, 5, 8, 16, 24, 100, 1000, 4099])
def test_widths(n):
    p = torch.randint(0, 4, (2, 4), device=DEV, generator=gen(n))
    check_states([state((2, 4, 3, n), torch.uint8), state((2, 4, n), torch.float32)], p)


def test_places_and_orders():
    x = state((2, 6, 8, 40), torch.float16)
    for p in ([0, 1, 2, 3, 4, 5], [5, 4, 3, 2, 1, 0], [1, 2, 3, 4, 5, 0], [0] * 6, [5] * 6, [1, 0, 3, 2, 5, 4], [-1, 6, 2 ** 31, -2 ** 40, 3, 3]):
        check_states([x.clone()], torch.tensor([p, p[::-1]], device=DEV))
    check_states([x.clone()], torch.randint(0, 6, (2, 6), device=DEV, generator=gen(51), dtype=torch.int32))
    check_states([x.clone()], torch.randint(0, 6, (2, 6), device=DEV, generator=gen(52)).short())
    check_states([x.clone()], torch.randint(0, 6, (6, 2), device=DEV, generator=gen(53)).t())


def test_leading_dimensions():
    check_states([state((4, 9), torch.float32)], torch.tensor([3, 3, 0, 1], device=DEV))
    check_states([state((2, 3, 4, 9), torch.float32)], torch.randint(0, 4, (2, 3, 4), device=DEV, generator=gen(54)))
    check_states([state((2, 0, 4, 9), torch.float32)], torch.zeros(2, 0, 4, dtype=torch.int64, device=DEV))
    check_states([state((2, 4, 0, 9), torch.float32)], torch.zeros(2, 4, dtype=torch.int64, device=DEV))
    one = state((3, 4, 9), torch.float32)
    p = torch.randint(0, 4, (3, 4), device=DEV, generator=gen(55))
    want = reordered(one, p)
    assert same(swvr_amd.reorder_beams(one, p), want)
    both = swvr_amd.reorder_beams((one, one), p)
    assert isinstance(both, tuple) and same(both[1], want)
    assert swvr_amd.reorder_beams([], p) == [] and swvr_amd.reorder_beams((), p, inplace=True) == ()
    assert swvr_amd.reorder_beams(one, p, inplace=True) is one and same(one, want)


def test_parts_of_caches():
    """Views of what is filled; the rest stays as it is."""
    p = torch.randint(0, 4, (3, 4), device=DEV, generator=gen(56))
    for part in (lambda x: x[:, :, :, :11], lambda x: x[:, :, :, 3:], lambda x: x[:, :, 1:3, 5:9, 2:5], lambda x: x[..., 0],
                 lambda x: x.transpose(2, 3), lambda x: x[:, :, :, :, ::2], lambda x: x[:, :, ::2, :, ::2]):
        cache = state((3, 4, 4, 17, 6), torch.bfloat16)
        before, want = cache.cpu().clone(), reordered(part(cache), p)
        assert same(swvr_amd.reorder_beams(part(cache), p), want)
        swvr_amd.reorder_beams(part(cache), p, inplace=True)
        part(before).copy_(want)
        assert same(cache, before)
    # keys and values side by side, and beams that are not next to each other
    cache = state((3, 4, 2, 5, 8), torch.float16)
    want = reordered(cache, p)
    swvr_amd.reorder_beams([cache[:, :, 0], cache[:, :, 1]], p, inplace=True)
    assert same(cache, want)
    cache = state((5, 3, 4, 8), torch.float16)       # positions first
    y = cache.permute(1, 2, 0, 3)
    want = reordered(y, p)
    swvr_amd.reorder_beams(y, p, inplace=True)
    assert same(y, want)


def test_a_list_of_all_sorts():
    p = torch.randint(0, 5, (2, 5), device=DEV, generator=gen(57))
    xs = [state((2, 5, 3, 16), torch.float16, i) for i in range(70)] + [state((2, 5, n), torch.int64, n) for n in (1, 2, 3)] + \
         [state((2, 5), torch.bool), state((2, 5, 3, 32), torch.float16)[..., :16]]
    check_states(xs, p)


def test_more_logits_than_32_bits_count():
    x = torch.empty(1, 256, 2 ** 21, dtype=torch.bfloat16, device=DEV).expand(5, 256, 2 ** 21)   # (views of one GB)
    x[0].normal_(generator=gen(90))
    s = -torch.rand(5, 256, device=DEV, generator=gen(91))
    want = swvr_amd.select_beams(x[:1], s[4:], 3)
    y = torch.empty(5 * 256, 2 ** 21, dtype=torch.bfloat16, device=DEV).view(5, 256, 2 ** 21)     # 2.7e9 logits
    y.copy_(x)
    assert all(torch.equal(a[4:], b) for a, b in zip(swvr_amd.select_beams(y, s, 3), want))


def test_offsets_past_32_bits():
    x = torch.empty(2, 3, 2 ** 30, dtype=torch.uint8, device=DEV)     # 6 GB
    for b in range(2):
        for w in range(3):
            x[b, w] = 16 * b + w + 1
    p = torch.tensor([[2, 2, 0], [1, 0, 1]], device=DEV)
    swvr_amd.reorder_beams(x, p, inplace=True)
    for b in range(2):
        for j in range(3):
            assert (x[b, j] == 16 * b + int(p[b, j]) + 1).all()


def test_lazy_views_and_versions():
    z = torch.randn(2, 3, 4, dtype=torch.complex64, device=DEV)
    p = torch.tensor([[1, 0, 2], [2, 2, 0]], device=DEV)
    for y in (z.conj(), z.conj().imag):
        assert torch.equal(swvr_amd.reorder_beams(y, p).cpu(), reordered(y, p))
        with pytest.raises(ValueError):
            swvr_amd.reorder_beams(y, p, inplace=True)
    x = torch.randn(2, 3, 4, device=DEV)
    leaf = torch.randn(2, 3, 4, device=DEV, requires_grad=True)
    loss = (leaf * x).sum()
    swvr_amd.reorder_beams(x, p, inplace=True)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    with torch.inference_mode():
        y = torch.randn(2, 3, 4, device=DEV)
        want = reordered(y, p)
        assert same(swvr_amd.reorder_beams(y, p, inplace=True), want)


def test_states_that_cannot_be_reordered_in_place():
    p = torch.zeros(2, 3, dtype=torch.int64, device=DEV)
    x = state((2, 3, 4), torch.float32)
    wide = state((2, 3, 4, 4, 4, 4, 4), torch.float32)[:, :, :3, :3, :3, :3, :3]
    for bad in ([x, x], [x, p], x[:, :1].expand(2, 3, 4), x[:1].expand(2, 3, 4), x[..., :1].expand(2, 3, 4), wide,
                state((20,), torch.float32).as_strided((2, 3, 4), (8, 2, 1)), state((3, 2, 2, 9), torch.float32)):
        with pytest.raises(ValueError):
            swvr_amd.reorder_beams(bad, p, inplace=True)
    assert same(swvr_amd.reorder_beams(wide, p), reordered(wide, p))
    assert same(swvr_amd.reorder_beams(x[:, :1].expand(2, 3, 4), p), reordered(x[:, :1].expand(2, 3, 4), p))
    with pytest.raises(ValueError, match="no gradient"):
        swvr_amd.reorder_beams(x.clone().requires_grad_(True), p)
    with torch.no_grad():
        y = x.clone().requires_grad_(True)
        assert same(swvr_amd.reorder_beams(y, p), reordered(y, p))


def test_states_captured_and_replayed():
    p = torch.zeros(3, 4, dtype=torch.int64, device=DEV)
    xs = [state((3, 4, 6, 10), torch.bfloat16, i) for i in range(4)]
    swvr_amd.reorder_beams(xs, p)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        swvr_amd.reorder_beams(xs, p, inplace=True)
        new = swvr_amd.reorder_beams(xs, p)
    for i in range(3):
        for j, x in enumerate(xs):
            x.copy_(state(x.shape, x.dtype, 10 * i + j))
        p.copy_(torch.randint(0, 4, (3, 4), device=DEV, generator=gen(60 + i)))
        once = [reordered(x, p) for x in xs]
        twice = [reordered(x, p) for x in once]
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(same(a, b) for a, b in zip(xs, once)) and all(same(a, b) for a, b in zip(new, twice))


def test_states_as_traced_and_compiled():
    p = torch.randint(0, 4, (2, 4), device=DEV, generator=gen(70))
    xs = [state((2, 4, 5, 8), torch.int32, i) for i in range(3)]
    torch.library.opcheck(torch.ops.swvr.reorder_beams.default, (xs, p), test_utils=("test_schema", "test_faketensor"))
    torch.library.opcheck(torch.ops.swvr.reorder_beams_.default, ([x.clone() for x in xs], p), test_utils=("test_schema", "test_faketensor"))
    want = [reordered(x, p) for x in xs]
    torch._dynamo.reset()
    got = torch.compile(lambda a, b: swvr_amd.reorder_beams(a, b * 1), fullgraph=True)(xs, p)
    assert all(same(a, b) for a, b in zip(got, want))

    def step(a, b):
        swvr_amd.reorder_beams(a, b * 1, inplace=True)
        return a[0] + 1

    torch._dynamo.reset()
    got = torch.compile(step, fullgraph=True)(xs, p)
    assert all(same(a, b) for a, b in zip(xs, want)) and same(got - 1, want[0])


# ---------------------------------------------------------------- together
def test_a_search():
    """Four steps of a search: the integers' logits, the best beams, their caches and tokens, the next inputs; each step
    against the definitions in 64 bits on what came before."""
    B, W, V, K = 3, 4, 517, 64
    g = gen(80)
    E = torch.randn(V, K, device=DEV, generator=g).to(torch.bfloat16)
    w = int8.quantize_rows(torch.randn(V, K, device=DEV, generator=g) * 0.4)
    cache = [torch.zeros(B, W, 2, 6, K, dtype=torch.bfloat16, device=DEV) for _ in range(2)]
    history = torch.full((B, W, 6), -1, device=DEV)
    scores = torch.full((B, W), -math.inf, device=DEV)
    scores[:, 0] = 0
    finished = torch.zeros(B, W, dtype=torch.bool, device=DEV)
    lengths = torch.zeros(B, W, dtype=torch.int64, device=DEV)
    h = torch.randn(B, 1, K, device=DEV, generator=g).to(torch.bfloat16).expand(B, W, K)
    for t in range(4):
        logits = int8.head_logits(h, w, dtype=torch.float32)
        logits[..., 2] += 2.0       # ends come up
        tokens, parents, new = check(logits, scores, finished=finished, end_id=2, lengths=lengths, length_penalty=0.6)
        kept = [x.cpu().clone() for x in (*cache, history, finished, lengths)]
        swvr_amd.reorder_beams([x[:, :, :, :t] for x in cache], parents, inplace=True)
        history, finished, lengths = swvr_amd.reorder_beams([history, finished, lengths], parents)
        p = parents.cpu()
        for x, before in zip(cache, kept):
            want = before.clone()
            want[:, :, :, :t] = reordered(before[:, :, :, :t], p)
            assert same(x, want)
        assert all(same(a, reordered(b, p)) for a, b in zip((history, finished, lengths), kept[2:]))
        lengths = lengths + (~finished).long()
        finished = finished | (tokens == 2)
        history[:, :, t] = tokens
        x = swvr_amd.embedding_lookup(tokens, E)
        for c in cache:
            c[:, :, :, t] = x[:, :, None]
        h = (x.float() + sum(c.float().mean(dim=(2, 3)) for c in cache)).to(torch.bfloat16)
        scores = new
    assert (history[:, :, :4] >= 0).all() and (scores[:, :-1] >= scores[:, 1:]).logical_or(lengths[:, :-1] != lengths[:, 1:]).all()
