"""The C ABI of the learned-feature operators writes its results and workspaces and nothing beside them: every array that a call
writes lies between two guards, at every boundary that its element type allows."""
import ctypes as C

import pytest
import torch

from event_3dgs_amd import _lib

pytestmark = pytest.mark.gpu
DEV, GUARD, MARK = "cuda", 8192, 0xFF      # (0xFF..: NaN in each of the types)
TYPES = [torch.float32, torch.float16, torch.bfloat16]


class Buffers:
    """Arrays between guards, filled with the guards' bytes."""
    def __init__(self):
        self.held = []

    def __call__(self, nbytes, offset=0):
        t = torch.full((2 * GUARD + nbytes + 256,), MARK, dtype=torch.uint8, device=DEV)
        assert t.data_ptr() % 256 == 0
        self.held.append((t, GUARD + offset, GUARD + offset + nbytes))
        return C.c_void_p(t.data_ptr() + GUARD + offset)

    def view(self, k, dtype, shape):
        t, lo, hi = self.held[k]
        return t[lo:hi].clone().view(dtype).view(shape)

    def check(self):
        torch.cuda.synchronize()
        for k, (t, lo, hi) in enumerate(self.held):
            assert (t[:lo] == MARK).all() and (t[hi:] == MARK).all(), "buffer %d" % k


def run(rc):
    assert rc == 0, _lib.lib().e3dgs_last_error().decode()


def ptr(t):
    return C.c_void_p(t.data_ptr())


def randn(*shape, dtype=torch.float32):
    return torch.randn(shape, generator=torch.Generator().manual_seed(sum(shape))).to(DEV).to(dtype)


@pytest.mark.parametrize("code, dtype", list(enumerate(TYPES)))
@pytest.mark.parametrize("n, rows, dim", [(1, 1, 1), (3, 5, 7), (200, 70, 33), (256, 3, 1030), (257, 9, 20), (1500, 40, 66), (5000, 3000, 5),
                                          (20001, 37, 12), (20001, 3, 129), (300001, 100, 2), (2100001, 50, 1), (0, 9, 5)])
def test_embedding(hip_lib, code, dtype, n, rows, dim):
    size = torch.finfo(dtype).bits // 8
    index = (torch.arange(n, device=DEV) * 7919 % (rows + 2) - 1).int()          # (-1 and one past the table among them)
    table, d = randn(rows, dim, dtype=dtype), randn(max(n, 1), dim, dtype=dtype)
    for offset in (0, size, 8):
        b = Buffers()
        out = b(n * dim * size, offset)
        run(hip_lib.e3dgs_embedding_forward(n, rows, dim, ptr(index), 4, ptr(table), dim, code, 1.0, out, None))
        grad, scratch = b(rows * dim * size, offset), b(hip_lib.e3dgs_embedding_backward_scratch_bytes(n, rows, dim))
        run(hip_lib.e3dgs_embedding_backward(n, rows, dim, ptr(index), 4, ptr(d), dim, code, 1.0, grad, scratch, None))
        b.check()
        at = index.long().clamp(0, rows - 1)
        want = torch.where((index < 0).unsqueeze(1), 0.0, table[at].float())
        want[index >= rows] = float("nan")
        assert torch.equal(torch.nan_to_num(b.view(0, dtype, (n, dim)).float(), nan=9.0), torch.nan_to_num(want, nan=9.0))
        assert torch.isfinite(b.view(1, dtype, (rows, dim)).float()).all()


@pytest.mark.parametrize("code, dtype", list(enumerate(TYPES)))
@pytest.mark.parametrize("rows, dim", [(1, 1), (3, 7), (301, 48), (5003, 59), (1030, 300), (2000, 511), (300, 514), (17, 1030), (1025, 2052),
                                       (40, 4097), (1030, 8200), (9, 16390), (70, 40001), (0, 6)])
def test_layer_norm(hip_lib, code, dtype, rows, dim):
    size = torch.finfo(dtype).bits // 8
    x, d, w = randn(max(rows, 1), dim, dtype=dtype), randn(max(rows, 1), dim, dtype=dtype), randn(dim)
    for offset in (0, size, 8):
        b = Buffers()
        out, mean, rstd = b(rows * dim * size, offset), b(rows * 4, 4), b(rows * 4, 4)
        run(hip_lib.e3dgs_layer_norm_forward(rows, dim, ptr(x), dim, code, ptr(w), ptr(w), 0, 1e-5, out, mean, rstd, None))
        dx, dw, db = b(rows * dim * size, offset), b(dim * 4, 4), b(dim * 4, 4)
        scratch = b(hip_lib.e3dgs_layer_norm_backward_scratch_bytes(rows, dim))
        run(hip_lib.e3dgs_layer_norm_backward(rows, dim, ptr(d), dim, ptr(x), dim, code, ptr(w), 0, mean, rstd, dx, dw, db, scratch, None))
        b.check()
        for k in range(6):
            t = b.view(k, dtype if k in (0, 3) else torch.float32, (-1,)).float()
            assert torch.isfinite(t).all() and (t.abs() < 1e4).all(), k            # (all of it is written)


@pytest.mark.parametrize("code, dtype", list(enumerate(TYPES)))
@pytest.mark.parametrize("rows, classes, k, planes", [
    (1, 1, 1, False), (5, 9, 2, False), (301, 59, 3, False), (1030, 2100, 4, False), (1030, 5001, 4, False), (7, 3001, 70, False),
    (3, 20001, 5, False), (2, 140001, 9, False), (35, 9, 2, True), (301, 59, 9, True), (1024, 256, 3, True), (262144, 5, 2, True),
    (262145, 5, 7, True), (0, 9, 2, False)])
def test_distill(hip_lib, code, dtype, rows, classes, k, planes):
    size = torch.finfo(dtype).bits // 8
    n = max(rows, 1)
    z = randn(classes, n, dtype=dtype) if planes else randn(n, classes, dtype=dtype)
    t, ids = randn(n, k), torch.randint(-1, classes, (n, k), generator=torch.Generator().manual_seed(n)).int().to(DEV)
    strides = (1, n) if planes else (classes, 1)
    head = (rows, classes, k, ptr(z), *strides, code, ptr(t), k, 1, 0, ptr(ids), k, 1, 4, 2.0)
    for offset in (0, size, 8):
        for how in (0, 1, 2):
            b = Buffers()
            stats, row_loss, loss, grad = b((2 * rows + 1) * 4), b(rows * 4, 4), b(4, 4), b(rows * classes * size, offset)
            scratch = b(hip_lib.e3dgs_distill_scratch_bytes(rows))
            run(hip_lib.e3dgs_distill_forward(*head, how, stats, row_loss, loss, grad, *strides, scratch, None))
            stats2, again = b((2 * rows + 1) * 4), b(rows * classes * size, offset)
            run(hip_lib.e3dgs_distill_forward(*head, how, stats2, None, loss, None, 0, 0, scratch, None))
            run(hip_lib.e3dgs_distill_backward(*head, how, stats2, None, again, *strides, None))
            b.check()
            for j in (1, 2, 3, 6):
                v = b.view(j, dtype if j in (3, 6) else torch.float32, (-1,)).float()
                assert torch.isfinite(v).all() and (v.abs() < (1e7 if j == 2 else 1e3)).all(), (how, j)
            assert (b.view(3, dtype, (-1,)).float() - b.view(6, dtype, (-1,)).float()).abs().sum() <= 1e-2 * max(1, rows)
