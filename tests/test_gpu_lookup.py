"""embedding_lookup on the GPU against 64-bit sums: types, widths from one column to many passes, ids that
repeat, pad or lie outside the table, strides, streams, graphs and compilation.

Tolerances: a row of out is one product (scale rounded to fp32, the product rounded, then rounded to the type): half a
step of the type plus two of fp32, relative.  A row of the gradient adds n cotangents in fp32, at most n half steps
of fp32 times the sum of their magnitudes, in parts that are fp32 themselves, then is scaled and rounded likewise."""
import math

import pytest
import torch

import swvr_amd

pytestmark = pytest.mark.gpu
DEV = "cuda"
F32 = 2.0 ** -24
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24, torch.float64: 2.0 ** -53}


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def make(N, V, D, dtype, seed=0):
    g = gen(seed)
    E = torch.randn(V, D, device=DEV, generator=g, dtype=torch.float64).to(dtype)
    return E, torch.randint(0, V, (N,), device=DEV, generator=g), torch.randn(N, D, device=DEV, generator=g).to(dtype)


def want_out(ids, E, scale):
    ids = ids.long()
    there = (ids >= 0) & (ids < E.shape[0])
    rows = torch.cat([E.double(), E.new_zeros(1, E.shape[1])])[ids.clamp(0, E.shape[0])] * scale
    rows = torch.where((ids < 0)[..., None], torch.zeros_like(rows), rows)
    return torch.where(((ids >= 0) & ~there)[..., None], torch.full_like(rows, math.nan), rows)


def want_grad(ids, g, V, scale):
    """(gradient, tolerance), in 64 bits; fp64 cotangents are summed with their low parts, as integers cannot be."""
    ids, g = ids.reshape(-1).long(), g.reshape(-1, g.shape[-1]).double()
    ok = (ids >= 0) & (ids < V)
    z = torch.zeros(V, g.shape[1], dtype=torch.float64, device=DEV)
    total = z.clone().index_put_((ids[ok],), g[ok], accumulate=True) * scale
    mag = z.clone().index_put_((ids[ok],), g[ok].abs(), accumulate=True) * abs(scale)
    n = torch.zeros(V, dtype=torch.float64, device=DEV).index_put_((ids[ok],), torch.ones_like(ids[ok], dtype=torch.float64),
                                                                 accumulate=True)
    return total, mag, n[:, None]


def check(ids, E, g, scale=1.0):
    E = E.detach().requires_grad_(True)
    out = swvr_amd.embedding_lookup(ids, E, scale=scale)
    (gE,) = torch.autograd.grad(out, E, g)
    assert out.dtype == gE.dtype == E.dtype and gE.shape == E.shape and out.shape == (*ids.shape, E.shape[1])
    step = F32 if E.dtype != torch.float64 else 2.0 ** -53
    want = want_out(ids, E.detach(), scale)
    assert torch.equal(torch.isnan(out), torch.isnan(want))
    # below the smallest normal number n0 the type's values lie eps n0 apart, whatever the value: half of that is
    # tiny (fp16: 2^-14 2^-11 = 2^-25, half its smallest value 2^-24)
    tiny = torch.finfo(E.dtype).smallest_normal * HALF[E.dtype]
    bad = (out.double() - want).abs() > want.abs() * (HALF[E.dtype] + 3 * step) + tiny
    assert not bad.any()
    total, mag, n = want_grad(ids, g, E.shape[0], scale)
    half = HALF[E.dtype]
    # the 64-bit sums of fp64 cotangents are off by as much as the kernel's
    tol = total.abs() * half + mag * (n + 3) * step * (2 if E.dtype == torch.float64 else 1) * (1 + half)
    assert not ((gE.double() - total).abs() > tol + tiny).any()
    assert (gE[n[:, 0] == 0] == 0).all()
    return out, gE


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32, torch.float64])
@pytest.mark.parametrize("N,V,D", [(1, 1, 1), (1, 1000, 64), (7, 3, 5), (64, 256, 8), (65, 257, 33), (300, 1000, 100),
                                   (513, 511, 300), (1025, 70000, 16), (4096, 300, 130), (5000, 2049, 2050),
                                   (1500, 200000, 40), (2048, 1000, 1030), (2049, 1000, 1030)])
def test_types_and_sizes(dtype, N, V, D):
    E, ids, g = make(N, V, D, dtype, seed=N + D)
    check(ids, E, g, scale=1.0)
    check(ids, E, g, scale=math.sqrt(D) / 3)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("share", [0.3, 0.9, 1.0])
@pytest.mark.parametrize("N,D", [(40, 24), (300, 520), (2048, 40), (2049, 40), (3000, 72), (20000, 64), (70001, 9)])
def test_one_id_holds_most_tokens(dtype, share, N, D):
    """Segments over many runs, beginning and ending anywhere in one."""
    V = 1500
    E, ids, g = make(N, V, D, dtype, seed=N)
    hot = torch.rand(N, device=DEV, generator=gen(1)) < share
    for at in (0, 255, 256, 1499):
        check(torch.where(hot, at, ids), E, g)


@pytest.mark.parametrize("id_dtype", [torch.int64, torch.int32])
@pytest.mark.parametrize("N", [9000, 100003])
def test_few_ids_hold_half_the_tokens(id_dtype, N):
    """Ids as text has them, the frequent ones first: one workgroup's ids hold more tokens than it keeps at a time."""
    V = 30000
    E, _, g = make(N, V, 12, torch.bfloat16, seed=N)
    ids = (V ** torch.rand(N, device=DEV, generator=gen(4), dtype=torch.float64) - 1).to(id_dtype)
    check(torch.where(torch.rand(N, device=DEV, generator=gen(5)) < 0.1, -1, ids), E, g)


def test_several_ids_share_the_tokens():
    """Runs of equal ids of every length around the runs that are summed together."""
    lengths = [1, 7, 8, 9, 31, 32, 33, 63, 64, 65, 127, 500, 1023, 1024, 1025, 2100]
    for most in (130, 2100):              # in one launch, and in several
        ids = torch.cat([torch.full((n,), 3 * i, device=DEV) for i, n in enumerate(lengths) if n <= most])
        ids = ids[torch.randperm(ids.numel(), device=DEV, generator=gen(2))]
        g = torch.randn(ids.numel(), 40, device=DEV, generator=gen(3))
        check(ids, torch.randn(50, 40, device=DEV), g)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float64])
def test_padding_and_ids_outside_the_table(dtype):
    check_padding(*make(700, 300, 48, dtype))
    check_padding(*make(2700, 300, 48, dtype))


def check_padding(E, ids, g):
    check(torch.where(torch.rand(ids.numel(), device=DEV) < 0.4, -1, ids), E, g)
    check(torch.full_like(ids, -1), E, g)
    wild = ids.clone()
    wild[::7] = 300
    wild[3::7] = -(2 ** 62)
    wild[5::7] = 2 ** 40 + 5
    wild[6::7] = 2 ** 32 + 1  # 1, if it were cut to 32 bits
    check(wild, E, g)


def test_no_tokens_and_empty_tables():
    E = torch.randn(30, 8, device=DEV)
    _, gE = check(torch.zeros(0, dtype=torch.int64, device=DEV), E, torch.zeros(0, 8, device=DEV))
    assert (gE == 0).all()
    ids = torch.tensor([-1, -5], device=DEV)
    out, gE = check(ids, E[:0], torch.zeros(2, 8, device=DEV))
    assert gE.shape == (0, 8) and (out == 0).all()
    assert swvr_amd.embedding_lookup(ids, E[:, :0]).shape == (2, 0)


def test_id_types_shapes_and_strides():
    E, ids, g = make(24, 100, 40, torch.bfloat16)
    base, gE = check(ids, E, g)
    for x in (ids.int(), ids.short(), ids.to(torch.uint8)):
        o, ge = check(x, E, g)
        assert torch.equal(o, base) and torch.equal(ge, gE)
    o, ge = check(ids.view(2, 3, 4), E, g.view(2, 3, 4, 40))
    assert torch.equal(o.view(24, 40), base) and torch.equal(ge, gE)
    strided = torch.zeros(24, 3, dtype=torch.int64, device=DEV)
    strided[:, 1] = ids
    o, ge = check(strided[:, 1], E, g)
    assert torch.equal(o, base) and torch.equal(ge, gE)
    # the table's rows apart, its columns apart, and off a 16-byte border
    wide = torch.zeros(100, 97, dtype=E.dtype, device=DEV)
    for view in (wide[:, :40], wide[:, 1:41], wide[:, 10:90:2]):
        view.copy_(E)
        o, ge = check(ids, view, g)
        assert torch.equal(o, base) and torch.equal(ge, gE)
    o, _ = check(ids, E[:1].expand(100, 40), g)
    assert torch.equal(o, E[:1].expand(24, 40))
    # scalars
    assert torch.equal(swvr_amd.embedding_lookup(ids[5], E), base[5])


def test_cotangents_of_every_stride():
    E, ids, g = make(33, 60, 24, torch.float32)
    for x in (g[:1].expand(33, 24), torch.ones((), device=DEV).expand(33, 24), torch.randn(24, 33, device=DEV).t(),
              torch.randn(33, 50, device=DEV)[:, 3:27]):
        check(ids, E, x)
    E2 = E.clone().requires_grad_(True)
    swvr_amd.embedding_lookup(ids, E2).sum().backward()
    assert torch.equal(E2.grad.sum(), torch.tensor(33.0 * 24, device=DEV))


def test_ids_changed_before_the_backward_are_refused():
    E, ids, g = make(3000, 60, 8, torch.float32)
    out = swvr_amd.embedding_lookup(ids, E.requires_grad_(True))
    ids[0] += 1
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        torch.autograd.grad(out, E, g)


def test_backward_twice_and_compiled_backward_give_the_same():
    for n in (900, 2600):
        E, ids, g = make(n, 700, 24, torch.float32)
        out = swvr_amd.embedding_lookup(ids, E.requires_grad_(True))
        first = torch.autograd.grad(out, E, g, retain_graph=True)[0]
        assert torch.equal(torch.autograd.grad(out, E, g)[0], first)
        assert torch.equal(torch.ops.swvr.embedding_bwd(g, ids, 700, 1.0), first)


def test_gradient_against_differences():
    E, ids, _ = make(9, 6, 5, torch.float64)
    ids[2], ids[5] = -1, ids[0]
    assert torch.autograd.gradcheck(lambda e: swvr_amd.embedding_lookup(ids, e, scale=0.7), (E.requires_grad_(True),))


def test_the_same_on_every_run():
    E, ids, g = make(30000, 700, 64, torch.bfloat16)
    ids = torch.where(torch.rand(30000, device=DEV, generator=gen(4)) < 0.5, 3, ids)
    first = check(ids, E, g)[1]
    for _ in range(3):
        assert torch.equal(check(ids, E, g)[1], first)


def test_offsets_beyond_32_bits():
    """A table of 2.2 G elements: rows whose offsets, in elements and in bytes, pass 32 bits."""
    V, D = 550000, 4000
    E = torch.zeros(V, D, dtype=torch.bfloat16, device=DEV)
    ids = torch.tensor([0, 268434, 268435, 268436, 536870, 536871, 549999, 549999], device=DEV)
    E[ids] = torch.arange(8, device=DEV, dtype=torch.bfloat16)[:, None] + 1
    E.requires_grad_(True)
    out = swvr_amd.embedding_lookup(ids, E)
    assert torch.equal(out, E.detach()[ids])
    g = torch.arange(1, 9, device=DEV).to(torch.bfloat16)[:, None].expand(8, D).contiguous()
    (gE,) = torch.autograd.grad(out, E, g)
    assert torch.equal(gE[ids[:6]], g[:6]) and (gE[549999] == 15).all()
    assert int((gE != 0).any(dim=1).sum()) == 7


def test_another_stream():
    E, ids, g = make(500, 900, 64, torch.bfloat16)
    want, want_g = check(ids, E, g)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        out, gE = check(ids, E, g)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(out, want) and torch.equal(gE, want_g)


def test_captured_and_replayed():
    """Forward and backward in a graph, replayed with new ids and values between eager calls."""
    for n in (900, 2600):
        captured(*make(n, 500, 64, torch.bfloat16))


def captured(E, ids, g):
    E.requires_grad_(True)

    def step():
        out = swvr_amd.embedding_lookup(ids, E, scale=2.0)
        return out, torch.autograd.grad(out, E, g)[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, gE = step()
    for k in range(4):
        ids.copy_(torch.randint(-1, 500, ids.shape, device=DEV, generator=gen(k)) if k != 2 else torch.full_like(ids, 7))
        g.normal_(generator=gen(10 + k))
        graph.replay()
        torch.cuda.synchronize()
        e_out, e_gE = step()
        assert torch.equal(out, e_out) and torch.equal(gE, e_gE)


def test_compiled_whole():
    E, ids, g = make(100, 60, 32, torch.bfloat16)
    want, want_g = check(ids, E, g)
    E = E.detach().requires_grad_(True)
    out = torch.compile(lambda i, e: swvr_amd.embedding_lookup(i, e), fullgraph=True)(ids, E)
    (gE,) = torch.autograd.grad(out, E, g)
    assert torch.equal(out, want) and torch.equal(gE, want_g)
