"""Settings of sample_tokens per row at the ends of their types."""
import pytest
import torch

import swvr_amd

from .test_gpu_sample import check, gen

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("V", [700, 6000, 20011])
def test_top_k_far_below_zero_and_far_above_the_row(V):
    """Every k but the two small ones keeps all tokens: as without top_k, with and without other filters."""
    ks = torch.tensor([-2 ** 63, -2 ** 32 + 5, -2 ** 31 - 1, -1, 0, 2 ** 31, 2 ** 32 + 5, 2 ** 63 - 1, 5, 1], device=DEV)
    x = torch.randn(10, V, device=DEV, generator=gen(V))
    u = torch.rand(10, device=DEV, generator=gen(1))
    for kw in (dict(), dict(top_p=0.9), dict(min_p=0.05), dict(top_p=0.8, temperature=0.5)):
        token, logprob = swvr_amd.sample_tokens(x, u, top_k=ks, **kw)
        want, want_lp = swvr_amd.sample_tokens(x, u, **kw)
        assert torch.equal(token[:8], want[:8]) and torch.equal(logprob[:8], want_lp[:8])
    check(x, u, top_k=ks.clamp(0, V))
    assert torch.equal(swvr_amd.sample_tokens(x, u, top_k=ks)[0], swvr_amd.sample_tokens(x, u, top_k=ks.clamp(0, V))[0])
