"""Sizes whose launches would pass the 2^32 threads of one grid are refused on the host (no GPU): such a launch runs the
remainder alone, without an error."""
import ctypes

import pytest

from swvr_amd import _lib

P = ctypes.c_void_p(4096)


def fwd(N, K=16, V=8, D=4, dtype=_lib.BF16, nbytes=64):
    return _lib.load().swvr_fwd(dtype, N, K, V, D, P, K, P, K, P, D, None, 1.0, P, P, P, nbytes, None)


def fwd_active(N, K=16, V=8, D=4, dtype=_lib.BF16, nbytes=64):
    return _lib.load().swvr_fwd_active(dtype, dtype, dtype, N, K, V, D, P, K, P, K, P, D, None, 1.0, P, P, P, P, nbytes, None)


def bwd(N, K=16, V=8, D=4, dtype=_lib.BF16, gh=P, nbytes=64):
    return _lib.load().swvr_bwd(dtype, N, K, V, D, P, K, P, K, P, D, None, 1.0, P, P, P, P, 8192, gh, dtype if gh else 0,
                                P, dtype, P, dtype, None, P, nbytes, None)


def fwd64(N, K=16, V=8, D=4, chunk=8192, nbytes=64):
    return _lib.load().swvr_fwd_f64(N, K, V, D, P, K, P, K, P, D, None, 1.0, chunk, P, P, P, nbytes, None)


def bwd64(N, K=16, V=8, D=4, chunk=8192, nbytes=64):
    return _lib.load().swvr_bwd_f64(N, K, V, D, P, K, P, K, P, D, None, 1.0, P, P, P, P, chunk, P, P, P, None, P, nbytes, None)


def mse(N, nbytes=64):
    return _lib.load().swvr_mse_loss(N, 4, P, P, P, _lib.F32, 4, None, 0.0, 2, P, P, P, P, P, nbytes, None)


@pytest.mark.parametrize("fn,held,past", [
    (fwd, dict(N=2 ** 25, D=2 ** 10), dict(N=2 ** 27, D=2 ** 10)),           # passes of up to 256 columns
    (fwd_active, dict(N=2 ** 25), dict(N=2 ** 26)),
    (bwd, dict(N=2 ** 20, D=2048), dict(N=2 ** 20, D=4096)),                  # gO packed
    (bwd, dict(N=64, V=2 ** 22, D=4096), dict(N=64, V=2 ** 22, D=8192)),      # E packed
    (bwd, dict(N=2 ** 22, K=2 ** 11), dict(N=2 ** 22, K=2 ** 12)),            # gh written
    (fwd64, dict(N=2 ** 23), dict(N=2 ** 24)),
    (fwd64, dict(N=2 ** 20, D=2 ** 11), dict(N=2 ** 20, D=2 ** 12)),
    (bwd64, dict(N=2 ** 18, V=9000), dict(N=2 ** 19, V=9000)),
    (mse, dict(N=2 ** 27), dict(N=2 ** 28)),
])
def test_grids(fn, held, past):
    """The sizes that a grid holds go on to the check of the workspace."""
    assert fn(**held) == _lib.EWORKSPACE
    assert fn(**past) == _lib.EINVAL and b"2^32 threads" in _lib.load().swvr_last_error()


def test_gh_alone_needs_its_grid():
    assert bwd(N=2 ** 22, K=2 ** 12, gh=None) == _lib.EWORKSPACE
