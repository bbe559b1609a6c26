"""What lies directly before and behind the outputs, images and workspaces of the decoding operators stays as it is: the
C ABI on pieces of larger buffers that hold a pattern, of the sizes that the header asks for and no more."""
import ctypes

import pytest
import torch

from swvr_amd import _lib, int8, reorder_beams, select_beams

pytestmark = pytest.mark.gpu
DEV = "cuda"
PATTERN, ROOM = 0xA5, 1 << 16


class Piece:
    """``nbytes`` in the middle of a buffer that holds PATTERN everywhere."""

    def __init__(self, nbytes, shift=0):
        self.all = torch.full((ROOM + shift + nbytes + ROOM,), PATTERN, dtype=torch.uint8, device=DEV)
        self.nbytes, self.at = nbytes, ROOM + shift
        self.address = self.all.data_ptr() + self.at

    def of(self, dtype, *shape):
        x = self.all[self.at:self.at + self.nbytes]
        return x.clone().view(dtype).reshape(shape)      # (a copy: a piece may begin at any element)

    def alone(self):
        return bool((self.all[:self.at] == PATTERN).all() and (self.all[self.at + self.nbytes:] == PATTERN).all())


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def run(name, *args):
    lib = _lib.load()
    _lib.call(getattr(lib, name), torch.device(DEV, torch.cuda.current_device()), *args)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("R,K", [(1, 1), (7, 1000), (8, 1024), (9, 1025), (255, 4096), (256, 64), (257, 65), (2047, 1100),
                                 (2049, 1100), (2048, 4096), (2305, 4097), (2050, 8193), (40, 8193)])
def test_images(R, K, dtype):
    lib = _lib.load()
    x = torch.randn(R, K, device=DEV, generator=gen(R)).to(dtype)
    image, scale, out = Piece(lib.swvr_int8_size(R, K)), Piece(4 * R), Piece(4 * R * K)
    run("swvr_int8_quantize", _lib.DTYPE_TAG[dtype], R, K, x.data_ptr(), K, image.address, scale.address)
    run("swvr_int8_unpack", R, K, image.address, scale.address, out.address)
    w = int8.quantize_rows(x)
    assert torch.equal(image.of(torch.int8, *w.q.shape), w.q) and torch.equal(scale.of(torch.float32, R), w.scale)
    assert torch.equal(out.of(torch.float32, R, K), int8.dequantize(w))
    assert image.alone() and scale.alone() and out.alone()
    q = torch.randint(-128, 128, (R, K), device=DEV, generator=gen(K), dtype=torch.int8)
    image = Piece(lib.swvr_int8_size(R, K))
    run("swvr_int8_pack", R, K, q.data_ptr(), K, image.address)
    assert torch.equal(image.of(torch.int8, *w.q.shape), int8.pack_rows(q, w.scale).q) and image.alone()


# tokens and rows one below, at and one past each kernel's tile, on few rows and on many; K past where 256 x 256 begin
@pytest.mark.parametrize("out_dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("K", [64, 1090])
@pytest.mark.parametrize("N,V", [(1, 1), (31, 33), (32, 31), (33, 63), (63, 129), (64, 65), (65, 127), (127, 129), (128, 64), (129, 640),
                                 (5, 30721), (32, 30848), (63, 15361), (64, 31104), (65, 30719), (129, 30721), (300, 15104),
                                 (300, 15105), (255, 20479), (257, 30849), (300, 21120), (511, 31105), (512, 31104)])
def test_logits(N, V, K, out_dtype):
    lib = _lib.load()
    E = torch.finfo(out_dtype).bits // 8
    h = torch.randn(N, K, device=DEV, generator=gen(N)).to(torch.bfloat16)
    w = int8.quantize_rows(torch.randn(V, K, device=DEV, generator=gen(V)).to(torch.bfloat16))
    want = int8.head_logits(h, w, dtype=out_dtype)
    need = lib.swvr_int8_logits_workspace_size(N, K)
    for shift in (0, E):        # (rows that may be whole lines, and ones that are not)
        out, ws = Piece(N * V * E, shift), Piece(need)
        run("swvr_int8_logits", _lib.BF16, _lib.DTYPE_TAG[out_dtype], N, K, V, h.data_ptr(), K, w.q.data_ptr(),
            w.scale.data_ptr(), None, 0, 1.0, out.address, ws.address, need)
        assert torch.equal(out.of(out_dtype, N, V), want)
        assert out.alone() and ws.alone()


@pytest.mark.parametrize("B,W,V,k", [(1, 1, 1, 1), (3, 4, 2, 4), (5, 4, 5001, 4), (2, 16, 700, 16), (2, 8, 2049, 32), (3, 8, 2048, 33),
                                     (2, 17, 130, 5), (1, 33, 9, 33), (2, 256, 40, 256), (1, 100, 515, 100), (3, 1, 300, 256)])
def test_selection(B, W, V, k):
    lib = _lib.load()
    x = torch.randn(B, W, V, device=DEV, generator=gen(V)).to(torch.bfloat16)
    for kept in (torch.float32, torch.float64):
        s = -torch.rand(B, W, device=DEV, generator=gen(W)).to(kept).cumsum(1)
        want = select_beams(x, s, k)
        need = lib.swvr_select_beams_workspace_size(B, W, V, k)
        e = torch.finfo(kept).bits // 8
        token, parent, score, ws = Piece(8 * B * k), Piece(8 * B * k), Piece(e * B * k), Piece(need)
        run("swvr_select_beams", _lib.BF16, B, W, V, k, x.data_ptr(), V, s.data_ptr(), int(kept == torch.float64), None, 0, None,
            0.0, token.address, parent.address, score.address, ws.address, need)
        got = token.of(torch.int64, B, k), parent.of(torch.int64, B, k), score.of(kept, B, k)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        assert all(p.alone() for p in (token, parent, score, ws))


@pytest.mark.parametrize("run_bytes", [1, 2, 12, 40, 256, 4112])
@pytest.mark.parametrize("W,k", [(1, 1), (3, 5), (4, 4), (8, 9), (17, 17), (40, 33), (5, 200)])
def test_states(W, k, run_bytes):
    B, n1, n2 = 3, 5, 2
    beam = run_bytes * n1 * n2
    x = torch.randint(0, 256, (B, W, n2, n1, run_bytes), device=DEV, generator=gen(k), dtype=torch.uint8)
    parents = torch.randint(-1, W + 1, (B, k), device=DEV, generator=gen(W))
    out = [Piece(B * k * beam, shift) for shift in (0, 1)]
    src = (ctypes.c_void_p * 2)(x.data_ptr(), x.data_ptr())
    dst = (ctypes.c_void_p * 2)(*(p.address for p in out))
    steps = (ctypes.c_int64 * 4)(W * beam, beam, run_bytes * n1, run_bytes)
    to = (ctypes.c_int64 * 4)(k * beam, beam, run_bytes * n1, run_bytes)
    run("swvr_reorder_beams", 2, src, dst, B, W, k, parents.data_ptr(), 1, run_bytes, n1, n2, steps, to)
    want = reorder_beams(x, parents)
    for p in out:
        assert torch.equal(p.of(torch.uint8, B, k, n2, n1, run_bytes), want) and p.alone()
