"""The token operators as custom ops, where tracing relies on what their fake versions say: shapes, types and strides of
real outputs, for hidden sizes that are padded and parameters of any layout."""
import pytest
import torch

import swvr_amd

from .test_gpu_distill import check, make

pytestmark = pytest.mark.gpu
DEV = "cuda"


def layouts(h, W, b):
    """(name, h, W, bias): dense, transposed, rows apart, a bias with a stride."""
    apart = torch.zeros(W.shape[0], W.shape[1] + 24, dtype=W.dtype, device=DEV)[:, :W.shape[1]].copy_(W)
    return [("dense", h, W, b), ("transposed", h.t().contiguous().t(), W.t().contiguous().t(), b),
            ("apart", h, apart, torch.stack([b, b], dim=1)[:, 0])]


@pytest.mark.parametrize("K", [64, 100])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_distill_ops_as_traced(K, dtype):
    h, W, b, t, ids = make(60, K, 300, 5, dtype)
    for _, h2, W2, b2 in layouts(h, W, b):
        xs = [x.detach().requires_grad_(True) for x in (h2, W2, b2)]
        args = (*xs, t, ids, None, 1.5, 1e-3, 2, 1.0, 8192, dtype, True)
        torch.library.opcheck(torch.ops.swvr.distill.default, args, test_utils=("test_schema", "test_faketensor"))
        loss, kept, sb = torch.ops.swvr.distill(*args)
        back = (torch.ones_like(loss), h2, W2, b2, ids, kept.detach(), sb.detach(), 1.5, 1e-3, 2, 1.0, 8192, dtype, True, True, True)
        torch.library.opcheck(torch.ops.swvr.distill_bwd.default, back, test_utils=("test_schema", "test_faketensor"))


@pytest.mark.parametrize("K", [64, 100])
def test_distill_compiled_on_any_layout(K):
    h, W, b, t, ids = make(200, K, 900, 6, torch.bfloat16)
    for _, h2, W2, b2 in layouts(h, W, b):
        want, want_g = check(h2, W2, b2, t, ids, chunk_size=8192)
        xs = [x.detach().requires_grad_(True) for x in (h2, W2, b2)]
        torch._dynamo.reset()
        f = torch.compile(lambda a, c, d: swvr_amd.softmax_distill(a * 2, c * 1, t, ids, d, logit_scale=0.5), fullgraph=True)
        loss = f(*xs)
        assert torch.equal(loss.detach(), want)
        gh, gW, gb = torch.autograd.grad(loss, xs)
        # (h doubled and the scale halved: powers of two, the same bits)
        assert torch.equal(gh, want_g[0]) and torch.equal(gW, want_g[1]) and torch.equal(gb, want_g[2])


def test_lookup_and_sample_ops_as_traced():
    E = torch.randn(90, 33, device=DEV).to(torch.bfloat16)
    ids = torch.randint(-1, 90, (4, 7), device=DEV)
    for table in (E, E.t().contiguous().t()):
        torch.library.opcheck(torch.ops.swvr.embedding.default, (ids, table, 2.0), test_utils=("test_schema", "test_faketensor"))
    g = torch.randn(4, 7, 33, device=DEV).to(torch.bfloat16)
    for cot in (g, g.transpose(0, 1).contiguous().transpose(0, 1)):
        torch.library.opcheck(torch.ops.swvr.embedding_bwd.default, (cot, ids, 90, 2.0), test_utils=("test_schema", "test_faketensor"))
    x, u = torch.randn(4, 7, 500, device=DEV), torch.rand(7, 4, device=DEV).t()
    torch.library.opcheck(torch.ops.swvr.sample.default, (x, u, 1.0, 0, 0.9, 0.0, None, None, None, None),
                          test_utils=("test_schema", "test_faketensor"))


def test_lookup_and_sample_compiled_on_any_layout():
    E, ids = torch.randn(90, 33, device=DEV).to(torch.bfloat16), torch.randint(-1, 90, (50,), device=DEV)
    g = torch.randn(50, 33, device=DEV).to(torch.bfloat16)
    for table, cot in ((E, g), (E.t().contiguous().t(), g.t().contiguous().t())):
        x = table.detach().requires_grad_(True)
        (want_g,) = torch.autograd.grad(swvr_amd.embedding_lookup(ids, x, scale=2.0), x, cot)
        torch._dynamo.reset()
        out = torch.compile(lambda i, e: swvr_amd.embedding_lookup(i, e * 2), fullgraph=True)(ids, x)
        assert torch.equal(out, swvr_amd.embedding_lookup(ids, table, scale=2.0))
        (gE,) = torch.autograd.grad(out, x, cot * 1)
        assert torch.equal(gE, want_g)
    x, u = torch.randn(4, 7, 500, device=DEV), torch.rand(7, 4, device=DEV).t()
    want = swvr_amd.sample_tokens(x, u, top_p=0.9)
    torch._dynamo.reset()
    got = torch.compile(lambda a, c: swvr_amd.sample_tokens(a * 1, c * 1, top_p=0.9), fullgraph=True)(x, u)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_transforms_are_right_or_refused():
    """Forward mode finds no rule on the ops, and a tangent is never dropped in silence; vmap calls them item by item."""
    import torch.autograd.forward_ad as fwd
    h, W, b, t, ids = make(20, 64, 90, 4, torch.float32)
    E, at = torch.randn(90, 8, device=DEV), torch.randint(0, 90, (5,), device=DEV)
    target, u = torch.randn(20, 8, device=DEV), torch.full((90,), 0.5, device=DEV)
    weight = torch.ones(20, device=DEV)
    calls = [(lambda x: swvr_amd.softmax_distill(x, W, t, ids, b), h),
             (lambda x: swvr_amd.softmax_distill(x, W, t, ids, b, reduction="none"), h),
             (lambda x: swvr_amd.embedding_lookup(at, x), E),
             (lambda x: swvr_amd.softmax_readout(x, W, E, b)[0], h),
             (lambda x: swvr_amd.softmax_readout_mse(x, W, E, target, b), h),
             (lambda x: swvr_amd.softmax_readout_mse(x, W, E, target, b, weight=weight), h)]
    errors = (RuntimeError, NotImplementedError)
    for call, x in calls:
        with fwd.dual_level():
            for y in (x, x.detach().requires_grad_(True)):
                with pytest.raises(errors):
                    call(fwd.make_dual(y, torch.ones_like(y)))
            call(x)                                        # (a level without a tangent is no matter)
        with pytest.raises(errors):
            torch.func.jvp(call, (x,), (torch.ones_like(x),))
        both = torch.func.vmap(call)(torch.stack([x, x * 2]))
        for got, y in zip(both, (x, x * 2)):
            want = call(y)
            assert torch.allclose(got, want, rtol=1e-5, atol=1e-6)
    with fwd.dual_level(), pytest.raises(errors):          # the loss's target
        swvr_amd.softmax_readout_mse(h, W, E, fwd.make_dual(target, torch.ones_like(target)), b)
    # sampling has no derivative
    sample = lambda x: swvr_amd.sample_tokens(x, u)
    with fwd.dual_level():
        token, logprob = sample(fwd.make_dual(E, torch.ones_like(E)))
        assert fwd.unpack_dual(logprob).tangent is None
    assert torch.equal(token, sample(E)[0])
    tokens, _ = torch.func.vmap(sample)(torch.stack([E, -E]))
    assert torch.equal(tokens[0], token) and torch.equal(tokens[1], sample(-E)[0])
