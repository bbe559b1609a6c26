"""swvr_int8_logits refuses operands that do not begin at an element (nothing is launched)."""
import ctypes

import pytest

from swvr_amd import _lib

A = ctypes.c_void_p(4096)


@pytest.mark.parametrize("dtype,out_dtype,b_dtype", [(_lib.BF16, _lib.F16, _lib.F32), (_lib.F32, _lib.F32, _lib.BF16)])
@pytest.mark.parametrize("name,at", [("h", 4097), ("out", 4097), ("bias", 4097), ("scale", 4098)])
def test_elements(dtype, out_dtype, b_dtype, name, at):
    p = {**dict(h=A, out=A, bias=A, scale=A), name: ctypes.c_void_p(at)}
    lib = _lib.load()
    assert lib.swvr_int8_logits(dtype, out_dtype, 4, 16, 9, p["h"], 16, A, p["scale"], p["bias"], b_dtype, 1.0, p["out"], A, 1 << 40,
                                None) == _lib.EINVAL
    assert b"aligned to their elements" in lib.swvr_last_error()
