"""Limits of the token operators that the host checks (no GPU): settings and sizes past which the kernels' arithmetic
would overflow are refused, in Python and by the C ABI, and nothing is launched."""
import pytest
import torch

import swvr_amd
from swvr_amd import _lib
from swvr_amd.tokens import _per_row

from .test_tokens_host import distill, distill_abi, distill_bwd_abi, embedding, embedding_bwd


@pytest.mark.parametrize("tau", [1e-45, 1e-39, 3e-39, 3.2e38])
def test_temperatures_whose_reciprocal_overflows(tau):
    with pytest.raises(ValueError, match="temperature"):
        distill(temperature=tau)
    for fn in (distill_abi, distill_bwd_abi):
        assert fn(tau=tau) == _lib.EINVAL
        assert b"temperature" in _lib.load().swvr_last_error()


@pytest.mark.parametrize("tau", [5e-39, 1e-30, 1e30])
def test_temperatures_in_range(tau):
    """(past the check of the temperature: these sizes are refused for their workspace)"""
    with pytest.raises(RuntimeError, match="AMD GPUs"):
        distill(temperature=tau)
    for fn in (distill_abi, distill_bwd_abi):
        assert fn(tau=tau, nbytes=64) == _lib.EWORKSPACE


def test_top_k_of_any_integer_type_keeps_its_meaning():
    """As the kernels get it, in 32 bits: 0 or less is all, and so is 2^31 - 1, the most that V can be."""
    most = 2 ** 31 - 1
    wide = torch.tensor([-2 ** 63, -2 ** 32 + 5, -2 ** 31 - 1, -1, 0, 7, most, 2 ** 31, 2 ** 32 + 5, 2 ** 63 - 1])
    got = _per_row(wide, torch.int32, 10)
    assert got.dtype == torch.int32 and got.tolist() == [0, 0, 0, 0, 0, 7, most, most, most, most]
    assert _per_row(torch.tensor([-5, 0, 200, 32767]).short(), torch.int32, 4).tolist() == [0, 0, 200, 32767]
    assert _per_row(torch.tensor([255, 3], dtype=torch.uint8), torch.int32, 2).tolist() == [255, 3]
    for dtype, x in ((torch.uint32, 2 ** 32 - 1), (torch.uint64, 2 ** 32 + 5), (torch.uint64, 2 ** 64 - 1)):
        got = _per_row(torch.tensor([x, 9], dtype=dtype), torch.int32, 2).tolist()
        assert got[0] in (0, most) and got[1] == 9, (dtype, x, got)   # all of them, either way


MOST = 2 ** 30


@pytest.mark.parametrize("size", [MOST + 1, 2 ** 31 - 256, 2 ** 31 - 2, 2 ** 31 - 1])
def test_tables_past_the_kernels_32_bit_steps(size):
    """Odd widths next to 2^31 would step past it in 32 bits, and the rows' borders too: both are refused."""
    lib = _lib.load()
    for fn in (embedding, embedding_bwd):
        for kw in (dict(D=size, lde=size) if fn is embedding else dict(D=size, ldg=size), dict(V=size)):
            assert fn(**kw) == _lib.EINVAL and b"bad sizes" in lib.swvr_last_error(), kw
    assert lib.swvr_embedding_sorted_size(5000, size) == 0
    for args in ((_lib.BF16, 5000, size, 4), (_lib.BF16, 5000, 4, size)):
        assert lib.swvr_embedding_bwd_workspace_size(*args) == 0


def test_the_largest_tables():
    """(past the check of the sizes: refused for what is missing)"""
    lib = _lib.load()
    assert embedding(V=MOST, E=None) == _lib.EINVAL and b"non-null" in lib.swvr_last_error()
    assert embedding(D=MOST, lde=MOST, E=None) == _lib.EINVAL and b"non-null" in lib.swvr_last_error()
    for kw in (dict(V=MOST), dict(D=MOST, ldg=MOST)):
        assert embedding_bwd(nbytes=16, **kw) == _lib.EWORKSPACE
    # order, ids and segments; a part in fp32 at each of two ends of 32 (N = 4000: 16) tokens' runs
    assert lib.swvr_embedding_sorted_size(4000, MOST) == 4 * (2 * 4000 + MOST + 1)
    assert lib.swvr_embedding_bwd_workspace_size(_lib.BF16, 4000, 4, MOST) >= 250 * 2 * MOST * 4


def test_more_tokens_than_a_grid_of_waves():
    for fn in (distill_abi, distill_bwd_abi):
        assert fn(N=2 ** 26, T=1) == _lib.EINVAL and b"bad sizes" in _lib.load().swvr_last_error()
        assert fn(N=2 ** 26 - 1, T=1, nbytes=64) == _lib.EWORKSPACE


@pytest.mark.parametrize("V", [MOST + 1, 2 ** 31 - 200, 2 ** 31 - 2])
def test_vocabularies_past_the_kernels_32_bit_steps(V):
    for fn in (distill_abi, distill_bwd_abi):
        assert fn(V=V) == _lib.EINVAL and b"bad sizes" in _lib.load().swvr_last_error()
        assert fn(V=MOST, nbytes=64) == _lib.EWORKSPACE
    assert _lib.load().swvr_distill_scores_size(_lib.BF16, _lib.BF16, 1, 2048, V, 2048) == 0
