"""Launch timing counts the decoding operators' launches under names of their own."""
import pytest
import torch

from swvr_amd import _lib, int8, reorder_beams, select_beams

pytestmark = pytest.mark.gpu


def test_each_operator_under_its_name():
    x = torch.randn(2, 3, 500, device="cuda")
    W = torch.randn(500, 64, device="cuda")
    h, q, parents = torch.randn(6, 64, device="cuda"), torch.zeros(9, 16, dtype=torch.int8, device="cuda"), torch.zeros(2, 3, device="cuda").long()
    _lib.kernel_timing(True)
    _lib.kernel_timing(None)
    try:
        w = int8.quantize_rows(W)
        int8.dequantize(w)
        int8.pack_rows(q, torch.ones(9, device="cuda"))
        int8.head_logits(h, w)       # (h's rows too)
        select_beams(x, x[..., 0], 2)
        reorder_beams(x, parents)
        torch.cuda.synchronize()
        counts = {name: n for name, (_, n) in _lib.kernel_timing(None).items()}
    finally:
        _lib.kernel_timing(False)
    assert counts == {"int8_rows": 4, "int8_logits": 1, "select_beams": 1, "reorder_beams": 1}
