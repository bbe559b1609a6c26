"""Logits whose scales lie far from 1: the product of logit_scale, a token's scale and a row's may leave fp32 where the
logit does not, or where the sum is 0 and the logit is the bias.

With u = 2^-24 a logit is off by 4 u of the product and u of the result (the roundings of the sum past 2^24, of two
products of scales and of the whole) and 2^-149 where it is denormal, then half a step of bf16."""
import math

import pytest
import torch

from swvr_amd import int8

pytestmark = pytest.mark.gpu
DEV = "cuda"
H_SIZES = [1.0, 1e36, 0.0, 1e-36, 1e20, 1.0, 1e-20, 1e30, 2e38, 1e-30, 1e-3]
W_SCALES = [1e-3, 1e4, 1e-38, 1.0, 1e-41, 1e36, 1e-30, 1e-3, 0.0, 1e25, 1e-20, -1e-3, -1e30]


def operands(N, V, K):
    """h in fp32 and a head, sizes of all kinds side by side; row 5 and every 37th of W are zeros."""
    g = torch.Generator(device=DEV).manual_seed(N + V)
    h = torch.randn(N, K, device=DEV, generator=g)
    h *= (0.4 * torch.tensor(H_SIZES, device=DEV).repeat(N // len(H_SIZES) + 1)[:N] / h.abs().amax(dim=1))[:, None]
    q = torch.randint(-127, 128, (V, K), device=DEV, generator=g, dtype=torch.int8)
    q[5 % V] = 0
    q[::37] = 0
    scale = torch.tensor(W_SCALES, device=DEV).repeat(V // len(W_SCALES) + 1)[:V]
    return h, q, scale, torch.randn(V, device=DEV, generator=g)


def check(h, q, scale, bias, c, dtype):
    got = int8.head_logits(h, int8.pack_rows(q, scale), bias, logit_scale=c, dtype=dtype).double()
    sh = torch.clamp(h.abs().amax(dim=1), min=1e-30) * torch.tensor(1.0, device=DEV).div(127)
    qh = (h.double() / sh.double()[:, None]).round()
    prod = (qh @ q.double().t()) * (sh.double() * c)[:, None] * scale.double()
    want = prod + (0.0 if bias is None else bias.double())
    u, info = 2.0 ** -24, torch.finfo(dtype)
    room = prod.abs() * 4 * u + want.abs() * u + 2.0 ** -149
    if dtype != torch.float32:
        room = room + want.abs() * info.eps / 2 * (1 + 2.0 ** -10)
    over = want.abs() > info.max * (1 + 2.0 ** -7)
    fine = want.abs() < info.max * (1 - 2.0 ** -7)
    assert torch.equal(got[over], want[over].sign() * math.inf)
    assert got[fine].isfinite().all()
    assert ((got - want).abs()[fine] <= room[fine]).all(), ((got - want).abs() / room)[fine].max()


# a size for each kernel: 32 and 64 tokens on few rows, then tiles of 128 x 64, 64 x 128, 128 x 128, 256 x 128, 256 x 256
FORMS = [(11, 500, 64), (40, 500, 64), (12, 31104, 64), (100, 500, 80), (300, 15000, 64), (300, 21120, 64), (500, 31104, 1030)]


@pytest.mark.parametrize("c", [1.0, -1e20, 1e-25])
@pytest.mark.parametrize("N,V,K", FORMS)
def test_scales_of_every_size(N, V, K, c):
    h, q, scale, bias = operands(N, V, K)
    for dtype in (torch.float32, torch.bfloat16):
        check(h, q, scale, bias, c, dtype)
    check(h, q, scale, None, c, torch.float32)


@pytest.mark.parametrize("N,V,K", FORMS)
def test_nothing_but_the_bias(N, V, K):
    """Rows of zeros under scales whose product leaves fp32."""
    h = torch.full((N, K), 1e36, device=DEV)
    w = int8.pack_rows(torch.zeros(V, K, dtype=torch.int8, device=DEV), torch.full((V,), 1e4, device=DEV))
    bias = torch.randn(V, device=DEV)
    for c in (1.0, 1e30):
        assert torch.equal(int8.head_logits(h, w, bias, logit_scale=c), bias.expand(N, V))
    assert (int8.head_logits(h, w) == 0).all()


@pytest.mark.parametrize("N,V,K", FORMS)
def test_neighbours_do_not_matter(N, V, K):
    """A token and a row of ordinary size have the same logits beside far ones."""
    g = torch.Generator(device=DEV).manual_seed(N)
    h = torch.randn(N, K, device=DEV, generator=g)
    q = torch.randint(-127, 128, (V, K), device=DEV, generator=g, dtype=torch.int8)
    scale, bias = torch.rand(V, device=DEV, generator=g) * 1e-3, torch.randn(V, device=DEV, generator=g)
    want = int8.head_logits(h, int8.pack_rows(q, scale), bias, logit_scale=0.3)
    far_h, far_scale = h.clone(), scale.clone()
    far_h[1::5] *= 1e36
    far_h[2::5] = 0
    far_scale[1::7], far_scale[3::7] = 1e20, 1e-38
    got = int8.head_logits(far_h, int8.pack_rows(q, far_scale), bias, logit_scale=0.3)
    rows, cols = torch.arange(N, device=DEV) % 5, torch.arange(V, device=DEV) % 7
    near = ((rows != 1) & (rows != 2))[:, None] & ((cols != 1) & (cols != 3))
    assert torch.equal(got[near], want[near])
