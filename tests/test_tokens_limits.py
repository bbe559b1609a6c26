"""Limits of the token operators that the host checks (no GPU): settings and sizes past which the kernels' arithmetic
would overflow are refused, in Python and by the C ABI, and nothing is launched."""
import pytest
import torch

import swvr_amd
from swvr_amd import _lib

from .test_tokens_host import distill, distill_abi, distill_bwd_abi


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
