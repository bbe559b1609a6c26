"""The head in integers on the GPU against its definition in 64 bits: quantisation with ties and rows of every kind,
logits for few and many tokens, odd sizes, types, strides, the longest reduction, graphs and compilation.

Integers are equal, scales too (one rounded product).  A logit is fma(float(sum), (logit_scale sh) sw, bias), so with u
= 2^-24 it is off by the roundings of the sum (past 2^24 alone), of logit_scale, of two products of scales and of the
whole: 4 u of the product and u of the result, then half a step of the result's type (fp16: no less than 2^-25, half its
smallest step)."""
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


def quantized(x):
    """(q, scale) by the definition, on the CPU."""
    x = x.detach().cpu()
    amax = x.float().abs().amax(dim=1)
    scale = torch.clamp(amax, min=1e-30) * torch.tensor(1.0, dtype=torch.float32).div(127)
    bad = ~x.isfinite().all(dim=1)
    scale = torch.where(bad, math.nan, scale)
    q = (x.double() / scale.double()[:, None]).round().nan_to_num(0.0)
    return torch.where(bad[:, None], 0.0, q), scale


def check_rows(x):
    w = int8.quantize_rows(x)
    q, scale = quantized(x)
    assert w.shape == tuple(x.shape) and w.scale.dtype == torch.float32
    assert torch.equal(w.scale.cpu().nan_to_num(-1.0), scale.nan_to_num(-1.0))
    fine = scale.isfinite()
    assert (q[fine].abs() <= 127).all()
    back = int8.dequantize(w).cpu()
    want = q.float() * scale[:, None]     # (one rounding of the same product)
    assert torch.equal(back[fine], want[fine]) and back[~fine].isnan().all()
    return w


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("R,K", [(1, 1), (3, 15), (31, 16), (33, 64), (257, 65), (700, 127), (8192, 100), (8500, 256), (5, 5000)])
def test_rows(R, K, dtype):
    check_rows((torch.randn(R, K, device=DEV, generator=gen(R + K)) * 0.02).to(dtype))


@pytest.mark.parametrize("dtype", TYPES)
def test_halves_go_to_even(dtype):
    """Rows whose largest is 127 2^e have whole steps of 2^e: halves are exact."""
    x = torch.cat([torch.arange(-126.5, 127, 1.0), torch.tensor([127.0, 0.5, -0.5, 1.5, 2.5])])
    rows = torch.stack([x * 2.0 ** e for e in (-3, 0, 2)]).to(DEV)
    if dtype == torch.bfloat16:   # (8 bits hold the halves up to 128)
        assert torch.equal(rows.to(dtype).float(), rows)
    check_rows(rows.to(dtype))
    check_rows(rows.to(dtype).repeat(3000, 1))


def test_quotients_next_to_a_half():
    """x one step of fp32 to either side of (n + 1/2) times the scale."""
    s = torch.tensor(0.7371, device=DEV)
    n = torch.arange(0, 126, device=DEV).float()
    mid = ((n + 0.5).double() * (s * 127 * (torch.tensor(1.0) / 127).item()).double()).float()
    up, down = torch.nextafter(mid, mid + 1), torch.nextafter(mid, mid - 1)
    row = torch.cat([(s * 127).reshape(1), mid, up, down, -mid, -up, -down])
    check_rows(torch.stack([row, row * 3.3, row * 1e-20, row * 1e20]))


@pytest.mark.parametrize("dtype", TYPES)
def test_rows_of_every_kind(dtype):
    x = torch.randn(300, 200, device=DEV, generator=gen(5)).to(dtype)
    x[1] = 0
    x[2, 7] = math.inf
    x[3, 150] = -math.inf
    x[4, 199] = math.nan
    x[5] = torch.finfo(dtype).max
    x[6] = torch.finfo(dtype).smallest_normal
    x[7] = torch.finfo(dtype).smallest_normal / 4
    x[8, 1:] = 0
    check_rows(x)
    check_rows(x.repeat(30, 1))   # (the form for many rows)


@pytest.mark.parametrize("dtype", TYPES)
def test_rows_of_any_layout(dtype):
    x = torch.randn(90, 77, device=DEV, generator=gen(6)).to(dtype)
    wide = torch.zeros(90, 100, dtype=dtype, device=DEV)
    wide[:, 3:80] = x
    for y in (x.t().contiguous().t(), wide[:, 3:80], x[:1].expand(50, 77), x[::2], x[:, ::2], x[:0]):
        check_rows(y)


def test_packed_integers_come_back():
    for R, K in ((1, 1), (40, 130), (300, 64), (257, 1000)):
        q = torch.randint(-128, 128, (R, K), device=DEV, generator=gen(R), dtype=torch.int8)
        for y in (q, q.t().contiguous().t(), torch.cat([q, q], dim=1)[:, 1:K + 1]):
            w = int8.pack_rows(y, torch.ones(R, device=DEV))
            assert torch.equal(int8.dequantize(w).to(torch.int8), y)
    scale = torch.rand(257, device=DEV, generator=gen(7)).double()
    w = int8.pack_rows(q, scale)
    scale.zero_()                 # (the handle's own)
    assert (w.scale > 0).any()


def check_logits(h, w, bias=None, logit_scale=1.0, dtype=None):
    out = int8.head_logits(h, w, bias, logit_scale=logit_scale, dtype=dtype)
    dtype = dtype or h.dtype
    V = w.shape[0]
    assert out.dtype == dtype and out.shape == (*h.shape[:-1], V) and out.is_contiguous()
    q, sh = quantized(h.reshape(-1, h.shape[-1]))
    if out.numel() == 0:
        return out
    # the rows' integers, from what they stand for
    W = (int8.dequantize(w).double() / w.scale.double()[:, None]).round().cpu()
    prod = (q @ W.t()) * (sh.double() * logit_scale)[:, None] * w.scale.cpu().double()
    want = prod + (bias.cpu().double() if bias is not None else 0.0)
    got = out.reshape(-1, V).cpu().double()
    u = 2.0 ** -24
    room = prod.abs() * 4 * u + want.abs() * u
    if dtype != torch.float32:
        room = room + want.abs() * torch.finfo(dtype).eps / 2 * (1 + 2.0 ** -10) + (2.0 ** -25 if dtype == torch.float16 else 0)
    fine = want.isfinite()
    assert (got.isfinite() == fine).all()
    assert ((got - want).abs()[fine] <= room[fine]).all(), ((got - want).abs() / room)[fine].max()
    return out


SIZES = [(1, 1, 1), (1, 1000, 64), (2, 31, 16), (5, 33, 63), (31, 257, 65), (32, 255, 256), (33, 300, 100), (64, 1000, 200),
         (65, 511, 64), (100, 4097, 320), (128, 256, 1000), (129, 33, 64), (256, 256, 64), (257, 1025, 129), (500, 700, 512),
         (1030, 258, 72)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N,V,K", SIZES)
def test_logits(N, V, K, dtype):
    g = gen(N + V + K)
    h = torch.randn(N, K, device=DEV, generator=g).to(dtype)
    w = int8.quantize_rows(torch.randn(V, K, device=DEV, generator=g) * K ** -0.5)
    bias = torch.randn(V, device=DEV, generator=g).to(dtype)
    check_logits(h, w)
    check_logits(h, w, bias, logit_scale=0.3, dtype=torch.float32)


# a size for each tile, with rows that share lines and rows of whole ones
@pytest.mark.parametrize("V", [0, 1])
@pytest.mark.parametrize("N,rows", [(3, 5000), (40, 9000), (5, 31104), (40, 16128), (100, 31104), (300, 21120), (300, 31104),
                                    (500, 31104), (200, 3000)])
def test_logits_of_every_tile(N, rows, V):
    V = rows - 103 * V
    h = torch.randn(N, 72, device=DEV, generator=gen(N)).to(torch.bfloat16)
    w = int8.quantize_rows(torch.randn(V, 72, device=DEV, generator=gen(V)))
    bias = torch.randn(V, device=DEV, generator=gen(V + 1))
    for dtype in (torch.bfloat16, torch.float32):
        check_logits(h, w, bias, dtype=dtype)


@pytest.mark.parametrize("K", [520, 1090])
@pytest.mark.parametrize("N,V", [(500, 31104), (250, 61441), (1100, 16127)])
def test_logits_of_the_largest_tile(N, V, K):
    h = torch.randn(N, K, device=DEV, generator=gen(N + 1)).to(torch.float16)
    w = int8.quantize_rows(torch.randn(V, K, device=DEV, generator=gen(V + 1)).to(torch.bfloat16))
    for dtype in (torch.float16, torch.float32):
        check_logits(h, w, torch.randn(V, device=DEV, generator=gen(V + 2)), dtype=dtype)


def test_more_values_than_32_bits_count():
    x = torch.randn(1000, 8192, device=DEV, generator=gen(40)).to(torch.bfloat16).repeat(300, 1)     # 2.5e9
    x[-1] *= 3
    w = int8.quantize_rows(x)
    last = int8.quantize_rows(x[-300:].clone())
    assert torch.equal(w.scale[-300:], last.scale)
    back = int8.dequantize(w)
    assert torch.equal(back[-300:], int8.dequantize(last)) and torch.equal(back[:1000], back[1000:2000])
    del x, back
    h = torch.randn(9000, 8192, device=DEV, generator=gen(41)).to(torch.bfloat16)                    # 2.7e9 logits
    out = int8.head_logits(h, w)
    for rows in (slice(0, 3), slice(8990, 9000)):
        assert torch.equal(out[rows], int8.head_logits(h[rows], w))


@pytest.mark.parametrize("out", TYPES)
@pytest.mark.parametrize("kind", TYPES + [torch.float64])
def test_types_of_the_bias_and_the_logits(kind, out):
    for N in (3, 300):
        h = torch.randn(N, 96, device=DEV, generator=gen(N)).to(torch.bfloat16)
        w = int8.quantize_rows(torch.randn(333, 96, device=DEV, generator=gen(9)))
        bias = torch.randn(333, 2, device=DEV, generator=gen(10)).to(kind)[:, 1]
        # (read as fp32)
        check_logits(h, w, bias.float() if kind == torch.float64 else bias, dtype=out)
        a, b = (int8.head_logits(h, w, x, dtype=out) for x in (bias, bias.float()))
        assert torch.equal(a, b)


def test_shapes_and_strides_of_h():
    w = int8.quantize_rows(torch.randn(130, 80, device=DEV, generator=gen(11)))
    h = torch.randn(4, 6, 80, device=DEV, generator=gen(12)).to(torch.bfloat16)
    wide = torch.zeros(4, 6, 96, device=DEV, dtype=torch.bfloat16)
    wide[..., 5:85] = h
    for x in (h, h[0, 0], h.transpose(0, 1), wide[..., 5:85], h[:1, :1].expand(3, 40, 80), h[:0], h[:, :0],
              h.transpose(1, 2).contiguous().transpose(1, 2)):
        check_logits(x, w)
    empty = int8.quantize_rows(torch.zeros(0, 80, device=DEV))
    assert int8.head_logits(h, empty).shape == (4, 6, 0)


@pytest.mark.parametrize("N", [1, 40, 300])
def test_the_longest_sums(N):
    """127 127 2^17 is below 2^31."""
    K = 2 ** 17
    h = torch.ones(N, K, device=DEV, dtype=torch.bfloat16)
    h[N // 2] = -1
    W = torch.ones(35, K, device=DEV, dtype=torch.float16)
    W[3, ::2] = -1
    check_logits(h, int8.quantize_rows(W), dtype=torch.float32)


@pytest.mark.parametrize("N", [4, 300])
def test_infinities_and_nan_stay_in_their_rows(N):
    h = torch.randn(N, 64, device=DEV, generator=gen(13))
    h[1, 3], h[2, 5] = math.inf, math.nan
    W = torch.randn(100, 64, device=DEV, generator=gen(14))
    W[7, 1], W[99, 63] = -math.inf, math.nan
    out = check_logits(h, int8.quantize_rows(W))
    bad = torch.zeros(N, 100, dtype=torch.bool, device=DEV)
    bad[1:3], bad[:, 7], bad[:, 99] = True, True, True
    assert torch.equal(out.isnan(), bad)
    bias = torch.zeros(100, device=DEV)
    bias[5] = -math.inf     # a masked token
    assert (int8.head_logits(h, int8.quantize_rows(W), bias)[3:, 5] == -math.inf).all()


def test_a_token_has_the_same_logits_in_any_call():
    h = torch.randn(600, 256, device=DEV, generator=gen(15)).to(torch.bfloat16)
    w = int8.quantize_rows(torch.randn(1001, 256, device=DEV, generator=gen(16)))
    bias = torch.randn(1001, device=DEV, generator=gen(17))
    whole = int8.head_logits(h, w, bias, logit_scale=0.7)
    for a, z in ((0, 1), (5, 37), (64, 128), (100, 220), (300, 600), (599, 600)):
        assert torch.equal(int8.head_logits(h[a:z], w, bias, logit_scale=0.7), whole[a:z])


def test_rows_behind_the_last_are_left():
    """Outputs and scratch of odd sizes among others: what lies around them stays."""
    h = torch.randn(300, 96, device=DEV, generator=gen(18)).to(torch.bfloat16)
    w = int8.quantize_rows(torch.randn(77, 96, device=DEV, generator=gen(19)))
    want = int8.head_logits(h, w)
    around = [torch.full((5000,), 7.0, device=DEV) for _ in range(20)]
    for n in (1, 17, 33, 65, 129, 299):
        assert torch.equal(int8.head_logits(h[:n], w), want[:n])
    assert all((x == 7).all() for x in around)


def test_captured_and_replayed():
    h = torch.randn(70, 128, device=DEV, generator=gen(20)).to(torch.bfloat16)
    w = int8.quantize_rows(torch.randn(999, 128, device=DEV, generator=gen(21)))
    graphs = []
    for n in (1, 70):
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            int8.head_logits(h[:n], w)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = int8.head_logits(h[:n], w)
        graphs.append((graph, out, n))
    for k in range(3):
        h.copy_(torch.randn(70, 128, device=DEV, generator=gen(30 + k)))
        torch.cuda.synchronize()
        for graph, _, _ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for _, out, n in graphs:
            assert torch.equal(out, int8.head_logits(h[:n], w))


def test_another_stream():
    h = torch.randn(40, 128, device=DEV, generator=gen(22)).to(torch.bfloat16)
    w = int8.quantize_rows(torch.randn(5000, 128, device=DEV, generator=gen(23)))
    want = int8.head_logits(h, w)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    outs = []
    for s in streams:
        with torch.cuda.stream(s):
            outs.append(int8.head_logits(h, w))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)


def test_as_traced_and_compiled():
    W = torch.randn(77, 100, device=DEV, generator=gen(24))
    h = torch.randn(3, 5, 100, device=DEV, generator=gen(25)).to(torch.bfloat16)
    bias = torch.randn(77, device=DEV)
    w = int8.quantize_rows(W)
    utils = ("test_schema", "test_faketensor")
    for x in (W, W.t().contiguous().t()):
        torch.library.opcheck(torch.ops.swvr.int8_quantize.default, (x,), test_utils=utils)
    q = torch.randint(-9, 9, (77, 100), device=DEV, dtype=torch.int8)
    for scale in (w.scale, w.scale.double(), torch.stack([w.scale, w.scale], dim=1)[:, 0]):
        torch.library.opcheck(torch.ops.swvr.int8_pack.default, (q, scale), test_utils=utils)
    torch.library.opcheck(torch.ops.swvr.int8_unpack.default, (w.q, w.scale, 77, 100), test_utils=utils)
    for x in (h, h.transpose(0, 1)):
        torch.library.opcheck(torch.ops.swvr.int8_logits.default, (x, w.q, w.scale, bias, 77, 0.5, torch.float32), test_utils=utils)
    want = int8.head_logits(h * 2, w, bias, dtype=torch.float32)
    torch._dynamo.reset()
    got = torch.compile(lambda a, b: int8.head_logits(a * 2, w, b, dtype=torch.float32), fullgraph=True)(h, bias)
    assert torch.equal(got, want)
    torch._dynamo.reset()
    packed = torch.compile(lambda a, b: int8.dequantize(int8.pack_rows(a, b)), fullgraph=True)(q, w.scale)
    assert torch.equal(packed, q.float() * w.scale[:, None])
    torch._dynamo.reset()
    back = torch.compile(lambda a: int8.dequantize(int8.quantize_rows(a * 1)), fullgraph=True)(W)
    assert torch.equal(back, int8.dequantize(w))


def test_calls_that_would_need_a_gradient_are_refused():
    h = torch.randn(3, 64, device=DEV, requires_grad=True)
    W = torch.randn(9, 64, device=DEV, requires_grad=True)
    w = int8.quantize_rows(W)
    with pytest.raises(ValueError, match="no gradient"):
        int8.head_logits(h, w)
    with torch.no_grad():
        check_logits(h, w)
    check_logits(h.detach(), w)
