"""Quantisation of many rows, and the logits of rows that were quantised so, against the definition in 64 bits.

2048 rows and more with K past 1024 take a wave a row: up to K = 4096 with 4 pieces of 16 values a lane, up to 8192 with
8, and beyond these the rest of the row in a second read; fewer rows take a workgroup each.  Integers are equal, scales
too (one rounded product), and so are the values that come back (one rounded product)."""
import math

import pytest
import torch

from swvr_amd import int8

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = [torch.bfloat16, torch.float16, torch.float32]
SIZES = [(2049, 1025), (2300, 2560), (2048, 4096), (2100, 4099), (2048, 8192), (2050, 8195), (2048, 9001),
         (2047, 1025), (2047, 8192), (1800, 8207), (300, 9001), (2500, 1024)]


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def definition(x):
    """(integers, scales) on the CPU, in 64 bits; a row that holds no number throughout has scale NaN and zeros."""
    x = x.cpu()
    bad = ~x.isfinite().all(dim=1)
    scale = x.abs().amax(dim=1).float().clamp_min(1e-30) * torch.ones((), dtype=torch.float32).div(127)
    q = (x.double() / scale.double()[:, None]).round()
    q[bad] = 0
    return q, torch.where(bad, math.nan, scale)


def integers(w):
    """The image's own bytes: [rows / 32][K / 64][values / 16][32 rows][16 values], rows padded to 256, K to 64."""
    R, K = w.shape
    y = w.q.cpu().reshape(w.q.shape[0], w.q.shape[1], 4, 32, 16).permute(0, 3, 1, 2, 4).reshape(w.q.shape[0] * 32, -1)
    assert (y[R:] == 0).all() and (y[:, K:] == 0).all()
    return y[:R, :K]


def check(x):
    w = int8.quantize_rows(x)
    q, scale = definition(x)
    assert torch.equal(w.scale.cpu().nan_to_num(-1.0), scale.nan_to_num(-1.0))
    assert torch.equal(integers(w).double(), q)
    fine = scale.isfinite()
    back = int8.dequantize(w).cpu()
    assert torch.equal(back[fine], (q.float() * scale[:, None])[fine]) and back[~fine].isnan().all()
    return w, q


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("R,K", SIZES)
def test_many_rows(R, K, dtype):
    x = torch.randn(R, K, device=DEV, generator=gen(R + K)).to(dtype)
    x[::3] *= 0.01
    x[1] = 0
    x[2, K - 1] = 30       # the largest at either end
    x[3, 0] = -30
    x[4, K - 1] = math.inf
    x[R - 1, K - 1] = math.nan
    x[R - 2, 0] = -math.inf
    x[5] = torch.arange(K, device=DEV).remainder(254).sub(126.5).to(dtype)      # halves exactly, in bf16 most
    x[5, K // 2] = 127
    check(x)


@pytest.mark.parametrize("R,K", [(2050, 8300), (2050, 20001), (2048, 2000)])
def test_where_rows_of_a_wave_are_no_numbers(R, K):
    """In the part of a row that is read twice, and in what is read once."""
    x = torch.randn(R, K, device=DEV, generator=gen(K)).to(torch.bfloat16)
    for i, at in enumerate((0, 1023, 1024, 4096, 8191, 8192, 8199, K - 1)):
        x[8 * i + 1, min(at, K - 1)] = math.inf
        x[8 * i + 2, min(at, K - 1)] = math.nan
    check(x)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("R,K", [(2049, 1025), (2048, 4097), (2060, 8200)])
def test_rows_at_strides(R, K, dtype):
    wide = torch.full((R, K + 7), 1e4, device=DEV, dtype=dtype)
    wide[:, 3:K + 3] = torch.randn(R, K, device=DEV, generator=gen(K)).to(dtype)
    check(wide[:, 3:K + 3])


@pytest.mark.parametrize("N,V,K,dtype", [(5, 2049, 1025, torch.bfloat16), (100, 2300, 2560, torch.float16),
                                         (40, 16128, 1090, torch.float32), (500, 31104, 1090, torch.bfloat16),
                                         (2100, 2050, 4099, torch.bfloat16), (2050, 2048, 8200, torch.float32)])
def test_logits_of_the_original_rows(N, V, K, dtype):
    """Integers of both operands from the matrices themselves.  A sum below 2^31 is rounded once past 2^24, products of
    scales twice, the whole once: 4 2^-24 of the product, 2^-24 of the logit."""
    W = torch.randn(V, K, device=DEV, generator=gen(V)).to(dtype)
    h = torch.randn(N, K, device=DEV, generator=gen(N)).to(dtype)
    bias = torch.randn(V, device=DEV, generator=gen(V + 1))
    got = int8.head_logits(h, int8.quantize_rows(W), bias, logit_scale=0.25, dtype=torch.float32)
    (qh, sh), (qw, sw) = definition(h), definition(W)
    prod = (qh.to(DEV) @ qw.to(DEV).t()) * (0.25 * sh.double().to(DEV))[:, None] * sw.double().to(DEV)
    want = prod + bias.double()
    assert ((got.double() - want).abs() <= prod.abs() * 4 * 2.0 ** -24 + want.abs() * 2.0 ** -24).all()
