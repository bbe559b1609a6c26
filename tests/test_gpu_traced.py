"""The readout as custom ops, compiled: what tracing was told of the outputs' strides holds for hidden sizes that are
padded and for parameters of any layout."""
import pytest
import torch

import swvr_amd

pytestmark = pytest.mark.gpu
DEV = "cuda"


def make(K, dtype):
    g = torch.Generator(device=DEV).manual_seed(K)
    r = lambda *s, sc=1.0: (sc * torch.randn(*s, device=DEV, generator=g)).to(dtype)
    return r(200, K), r(700, K, sc=K ** -0.5), r(700, 40), r(700)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32, torch.float64])
@pytest.mark.parametrize("K", [64, 100])
@pytest.mark.parametrize("transposed", [False, True])
def test_gradients_of_a_compiled_readout(dtype, K, transposed):
    h, W, E, b = make(K, dtype)
    if transposed:
        h, W, E = (x.t().contiguous().t() for x in (h, W, E))
    target, weight = torch.randn(200, 40, device=DEV), (torch.rand(200, device=DEV) > 0.3).float()

    def run(fn):
        xs = [x.detach().requires_grad_(True) for x in (h, W, E, b)]
        out = fn(*xs)
        return out.detach(), torch.autograd.grad(out, xs)

    for f in (lambda h, W, E, b: swvr_amd.softmax_readout(h, W, E, b, chunk_size=8192)[0].square().sum(),
              lambda h, W, E, b: swvr_amd.softmax_readout_mse(h, W, E, target, b, chunk_size=8192),
              lambda h, W, E, b: swvr_amd.softmax_readout_mse(h, W, E, target, b, weight=weight, chunk_size=8192)):
        want, want_g = run(f)
        torch._dynamo.reset()
        got, got_g = run(torch.compile(lambda h, W, E, b: f(h * 1, W * 1, E * 1, b), fullgraph=True))
        assert (got - want).abs() <= 1e-5 * want.abs()   # (the sum of squares is compiled too)
        for a, c in zip(got_g, want_g):
            assert a.shape == c.shape and a.dtype == c.dtype
            assert (a.double() - c.double()).norm() <= 1e-5 * c.double().norm() + 2 ** -8 * c.double().norm() * (dtype == torch.bfloat16)
