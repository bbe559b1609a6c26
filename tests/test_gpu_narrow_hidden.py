"""Hidden sizes of one or two K-slices with several token blocks per workgroup: the backward's stages of one block are
fewer than its ring is deep, so what a block's epilogue reads must outlive the loads of the blocks after it."""
import pytest
import torch

import swvr_amd

from .gpu_util import rel_err
from .test_gpu_distill import close, formula

pytestmark = pytest.mark.gpu
DEV = "cuda"


def make(N, K, V, D, dtype, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    r = lambda *s, sc=1.0: (sc * torch.randn(*s, device=DEV, generator=g)).to(dtype)
    return r(N, K), r(V, K, sc=2 * K ** -0.5), r(V, D), r(V, sc=0.5), r(N, D).float(), r(N).float()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("K", [1, 8, 31, 32, 33, 64, 65])
@pytest.mark.parametrize("D", [1, 16, 32, 33, 64, 65, 130])
@pytest.mark.parametrize("N,V", [(9000, 8500)])
def test_readout(dtype, K, D, N, V):
    """Norm-wise, as the parity tests hold it: 1e-5 for O and LSE in fp32, 2e-2 for gradients of 2-byte operands."""
    h, W, E, b, gO, gl = make(N, K, V, D, dtype)
    xs = [x.requires_grad_(True) for x in (h, W, E, b)]
    O, lse = swvr_amd.softmax_readout(*xs)
    got = torch.autograd.grad((O * gO).sum() + (lse * gl).sum(), xs)
    with torch.no_grad():
        hd, Wd, Ed, dO = h.double(), W.double(), E.double(), gO.double()
        S = hd @ Wd.t() + b.double()
        want_lse = torch.logsumexp(S, dim=1)
        P = torch.exp(S - want_lse[:, None])
        del S
        want_O = P @ Ed
        dS = dO @ Ed.t()
        dS += (gl.double() - (dO * want_O).sum(dim=1))[:, None]
        dS *= P
        want = (dS @ Wd, dS.t() @ hd, P.t() @ dO, dS.sum(dim=0))
    assert rel_err(lse, want_lse) < 1e-5 and rel_err(O, want_O) < (1e-5 if dtype == torch.float32 else 1e-2)
    for a, c in zip(got, want):
        assert rel_err(a, c) < (1e-4 if dtype == torch.float32 else 2e-2)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("K", [1, 8, 32, 40])
@pytest.mark.parametrize("N,V,weighted", [(9000, 8500, False), (9000, 8500, True), (70000, 300, False)])
def test_distill(dtype, K, N, V, weighted):
    """Element by element, to the tolerances of the arithmetic."""
    h, W, _, b, t, gl = make(N, K, V, 6, dtype)
    ids = torch.randint(-1, V, (N, 6), device=DEV, generator=torch.Generator(device=DEV).manual_seed(1))
    weight = (gl > -0.5).float() if weighted else None
    xs = [x.requires_grad_(True) for x in (h, W, b)]
    loss = swvr_amd.softmax_distill(h, W, t, ids, b, weight=weight, reduction="sum")
    grads = torch.autograd.grad(loss, xs)
    want, want_g, tol = formula(h.detach(), W.detach(), b.detach(), t, ids, weight=weight, reduction="sum")
    close(loss.detach(), want, tol["loss"])
    for name, got in zip("hWb", grads):
        close(got, want_g[name], tol[name])


def test_quantised_readout():
    """The e4m3 scores at one slice of K, which keep all of a block's side stages in LDS: the same on every run."""
    from swvr_amd import fp8
    h, W, E, b, gO, gl = make(9000, 32, 8500, 16, torch.bfloat16)
    runs = []
    for _ in range(3):
        xs = [x.detach().requires_grad_(True) for x in (h, W, E, b)]
        O, lse = fp8.softmax_readout_fp8(*xs)
        runs.append(torch.autograd.grad((O * gO).sum() + (lse * gl).sum(), xs))
    assert all(torch.equal(a, c) for r in runs[1:] for a, c in zip(r, runs[0]))
