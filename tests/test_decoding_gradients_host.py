"""The decoding operators have no derivatives: what carries a tangent, or would record a gradient where none is given
back, is refused (checked before the device is, so here without one)."""
import pytest
import torch
from torch.autograd import forward_ad

import swvr_amd
from swvr_amd import int8

X, S = torch.zeros(2, 3, 9), torch.zeros(2, 3)
P, C, H = torch.zeros(2, 3, dtype=torch.int64), torch.zeros(2, 3, 4, 5), torch.zeros(4, 16)
Q = torch.zeros(9, 16, dtype=torch.int8)


def rows(scale):
    return int8.Int8Rows(torch.zeros(int8._image_shape(9, 16), dtype=torch.int8), scale, (9, 16))


CALLS = {
    "select_beams, logits": (X, lambda x: swvr_amd.select_beams(x, S)),
    "select_beams, scores": (S, lambda s: swvr_amd.select_beams(X, s)),
    "reorder_beams": (C, lambda c: swvr_amd.reorder_beams(c, P)),
    "reorder_beams, a list": (C, lambda c: swvr_amd.reorder_beams([C, c], P)),
    "reorder_beams, in place": (C, lambda c: swvr_amd.reorder_beams(c, P, inplace=True)),
    "quantize_rows": (H, lambda h: int8.quantize_rows(h)),
    "pack_rows": (torch.zeros(9), lambda s: int8.pack_rows(Q, s)),
    "dequantize": (torch.zeros(9), lambda s: int8.dequantize(rows(s))),
    "head_logits, h": (H, lambda h: int8.head_logits(h, rows(torch.zeros(9)))),
    "head_logits, bias": (torch.zeros(9), lambda b: int8.head_logits(H, rows(torch.zeros(9)), b)),
    "head_logits, scales": (torch.zeros(9), lambda s: int8.head_logits(H, rows(s))),
}


@pytest.mark.parametrize("name", CALLS)
def test_tangents_are_refused(name):
    x, call = CALLS[name]
    with forward_ad.dual_level():
        with pytest.raises(NotImplementedError, match="forward-mode"):
            call(forward_ad.make_dual(x.clone(), torch.ones_like(x)))
        with pytest.raises(RuntimeError, match="AMD GPUs"):      # (a level alone is nothing to refuse)
            call(x)


@pytest.mark.parametrize("name", ["dequantize", "head_logits, h", "head_logits, bias", "head_logits, scales", "reorder_beams",
                                  "reorder_beams, a list", "reorder_beams, in place"])
def test_gradients_are_refused(name):
    x, call = CALLS[name]
    leaf = x.clone().requires_grad_(True)
    with pytest.raises(ValueError, match="no gradient"):
        call(leaf)
    with torch.no_grad(), pytest.raises(RuntimeError, match="AMD GPUs"):
        call(leaf)
