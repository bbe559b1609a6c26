"""The token operators past the threads of one grid (2^32), where a call takes several launches."""
import pytest
import torch

import swvr_amd

from .test_gpu_distill import close, formula

pytestmark = pytest.mark.gpu
DEV = "cuda"


def test_lookup_of_more_ids_than_a_grid_holds():
    """A workgroup per row of 233 two-byte vectors: 2^24 of them are 2^32 threads."""
    N, V, D = 2 ** 24 + 2 ** 22 + 5, 300, 233
    E = torch.randn(V, D, device=DEV, generator=torch.Generator(device=DEV).manual_seed(0)).to(torch.bfloat16)
    ids = (torch.arange(N, device=DEV, dtype=torch.int32) * 7) % V
    with torch.no_grad():
        out = swvr_amd.embedding_lookup(ids, E)
    for i in range(0, N, 2 ** 22):
        assert torch.equal(out[i:i + 2 ** 22], E[ids[i:i + 2 ** 22].long()])


@pytest.mark.parametrize("N", [50, 2100])       # in one launch, and sorted
def test_gradient_of_the_longest_table(N):
    """2^30 rows, most of them zero: 2^24 workgroups of zero rows beside the sums'."""
    V = 2 ** 30
    ids = torch.cat([torch.arange(20, device=DEV), V - 1 - torch.arange(20, device=DEV),
                     torch.randint(0, V, (N - 40,), device=DEV, generator=torch.Generator(device=DEV).manual_seed(1))])
    ids = torch.cat([ids[5:], ids[:5]])
    E = torch.zeros(V, 1, device=DEV, dtype=torch.bfloat16)
    E[ids] = torch.rand(N, 1, device=DEV).to(torch.bfloat16) + 1
    E.requires_grad_(True)
    out = swvr_amd.embedding_lookup(ids, E)
    assert torch.equal(out, E.detach()[ids])
    g = torch.randint(1, 5, (N, 1), device=DEV).to(torch.bfloat16)
    (gE,) = torch.autograd.grad(out, E, g)
    where, back = ids.unique(return_inverse=True)
    want = torch.zeros(where.numel(), 1, device=DEV).index_add_(0, back, g.float())   # small whole numbers: exact
    assert torch.equal(gE[where].float(), want)
    gE[where] = 0
    assert not gE.any()


def test_distill_of_more_entries_than_a_grid_holds():
    """2^28 + 2^12 entries, a wave for every 4: 2^32 threads and more.  Terms and h's gradient of the first tokens and
    of the last."""
    N, K, V, T = 2 ** 18 + 4, 8, 300, 1024
    g = torch.Generator(device=DEV).manual_seed(2)
    h = torch.randn(N, K, device=DEV, generator=g).to(torch.bfloat16)
    W = torch.randn(V, K, device=DEV, generator=g).to(torch.bfloat16)
    ids = torch.randint(-1, V, (1, T), device=DEV, generator=g).expand(N, T)
    t = torch.randn(1, T, device=DEV, generator=g).expand(N, T)
    x = h.detach().requires_grad_(True)
    loss = swvr_amd.softmax_distill(x, W, t, ids, reduction="none")
    (gh,) = torch.autograd.grad(loss, x, torch.ones(N, device=DEV))
    for rows in (slice(0, 300), slice(N - 300, N)):
        want, want_g, tol = formula(h[rows], W, None, t[rows], ids[rows], reduction="none")
        close(loss[rows].detach(), want, tol["loss"])
        close(gh[rows], want_g["h"], tol["h"])
