"""A beam's sums are the same bits whatever stands beside it and however many candidates are kept: the order in which a
row's pieces of 2048 logits are added depends on V alone, in the kernel that selects in one launch (up to 16 beams, 32
candidates each, 256 in all) as in those for larger searches."""
import math

import pytest
import torch

import swvr_amd

pytestmark = pytest.mark.gpu
DEV = "cuda"


def make(B, W, V, dtype):
    g = torch.Generator(device=DEV).manual_seed(V + W)
    x = (torch.randn(B, W, V, device=DEV, generator=g) * 3).to(dtype)
    x[..., : V // 50] = -math.inf
    x[:, :, V // 2: V // 2 + 4096] = -math.inf      # a piece without a candidate
    return x, -5 - torch.rand(B, W, device=DEV, generator=g, dtype=torch.float64).cumsum(1)


def same(a, b):
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    assert torch.equal(a[2].view(torch.int64), b[2].view(torch.int64))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("V", [5001, 131072, 131073, 151936, 300001, 2 ** 21])
def test_numbers_of_candidates(V, dtype):
    x, s = make(12, 8, V, dtype)
    best = swvr_amd.select_beams(x, s, 33)
    same(swvr_amd.select_beams(x, s, 32), [t[:, :32] for t in best])


@pytest.mark.parametrize("V", [5001, 131073, 151936, 300001, 2 ** 21])
def test_numbers_of_beams(V):
    x, s = make(5, 17, V, torch.float16)
    s[:, 16] = -math.inf
    lengths = torch.arange(85, device=DEV).reshape(5, 17)
    for kw in ({}, {"lengths": True, "length_penalty": 0.7}):
        def of(w):
            return swvr_amd.select_beams(x[:, :w], s[:, :w], 16, **{**kw, **({"lengths": lengths[:, :w]} if kw else {})})
        same(of(16), of(17))
