"""Arguments the learned-feature operators refuse, and what they need, without a GPU: every refusal comes from the host checks."""
import ctypes as C

import pytest
import torch

from event_3dgs_amd import _lib, features, losses

PTR = C.c_void_p(4096)          # never followed: the calls below are refused before anything is launched


def text():
    return _lib.lib().e3dgs_last_error().decode()


def test_cpu_tensors_are_refused():
    x = torch.zeros(3, 4)
    i = torch.zeros(3, 1, dtype=torch.int64)
    for call in (lambda: features.embedding(i, x), lambda: features.layer_norm(x), lambda: losses.distill_loss(x, x[:, :1], i),
                 lambda: losses.distill_loss_raw(x, x[:, :1], i)):
        with pytest.raises(RuntimeError, match="no CPU path"):
            call()


def test_unknown_reduction_is_refused():
    x = torch.zeros(3, 4)
    for call in (losses.distill_loss, losses.distill_loss_raw):
        with pytest.raises(ValueError, match="reduction"):
            call(x, x[:, :1], torch.zeros(3, 1, dtype=torch.int64), reduction="average")


@pytest.mark.parametrize("n, rows, dim, index_bytes, dtype, ptr", [
    (4, 8, 0, 4, 0, PTR), (4, 8, (1 << 20) + 1, 4, 0, PTR), (4, 1 << 31, 4, 4, 0, PTR), (1 << 31, 8, 4, 4, 0, PTR),
    (4, 8, 4, 2, 0, PTR), (4, 8, 4, 4, 3, PTR), (4, 8, 4, 4, -1, PTR), (4, 8, 4, 4, 0, None)])
def test_embedding_arguments(hip_lib, n, rows, dim, index_bytes, dtype, ptr):
    assert hip_lib.e3dgs_embedding_forward(n, rows, dim, PTR, index_bytes, PTR, dim, dtype, 1.0, ptr, None) != 0
    assert "e3dgs_embedding_forward" in text()
    assert hip_lib.e3dgs_embedding_backward(n, rows, dim, PTR, index_bytes, PTR, dim, dtype, 1.0, ptr, PTR, None) != 0
    assert "e3dgs_embedding_backward" in text()


def test_embedding_scratch(hip_lib):
    assert hip_lib.e3dgs_embedding_backward(4, 8, 4, PTR, 4, PTR, 4, 0, 1.0, PTR, C.c_void_p(4096 + 8), None) != 0
    assert "aligned" in text()
    small, large = (hip_lib.e3dgs_embedding_backward_scratch_bytes(n, 4096, 48) for n in (0, 1000000))
    assert 0 < small < large


@pytest.mark.parametrize("dim, eps, dtype, affine, ptr", [
    (0, 1e-5, 0, 0, PTR), ((1 << 20) + 1, 1e-5, 0, 0, PTR), (4, -1.0, 0, 0, PTR), (4, float("nan"), 0, 0, PTR),
    (4, 1e-5, 3, 0, PTR), (4, 1e-5, 0, 5, PTR), (4, 1e-5, 0, 0, None)])
def test_layer_norm_arguments(hip_lib, dim, eps, dtype, affine, ptr):
    assert hip_lib.e3dgs_layer_norm_forward(3, dim, ptr, dim, dtype, PTR, PTR, affine, eps, PTR, PTR, PTR, None) != 0
    assert "e3dgs_layer_norm_forward" in text()
    if eps == 1e-5:
        assert hip_lib.e3dgs_layer_norm_backward(3, dim, PTR, dim, ptr, dim, dtype, PTR, affine, PTR, PTR, PTR, PTR, PTR, PTR, None) != 0
        assert "e3dgs_layer_norm_backward" in text()


@pytest.mark.parametrize("change", [
    dict(classes=0), dict(classes=1 << 31), dict(k=0), dict(k=1025), dict(rows=1 << 31), dict(temperature=0.0),
    dict(temperature=float("nan")), dict(temperature=float("inf")), dict(reduction=3), dict(dtype=3), dict(teacher_dtype=-1),
    dict(index_bytes=2), dict(logits=None), dict(index=None),
    dict(row_stride=1, class_stride=5, classes=257), dict(row_stride=7, class_stride=5)])
def test_distill_arguments(hip_lib, change):
    a = dict(rows=5, classes=9, k=2, logits=PTR, row_stride=9, class_stride=1, dtype=0, teacher_dtype=0, index=PTR,
             index_bytes=4, temperature=1.0, reduction=1)
    a.update(change)
    head = (a["rows"], a["classes"], a["k"], a["logits"], a["row_stride"], a["class_stride"], a["dtype"], PTR, a["k"], 1,
            a["teacher_dtype"], a["index"], a["k"], 1, a["index_bytes"], a["temperature"], a["reduction"])
    assert hip_lib.e3dgs_distill_forward(*head, PTR, PTR, PTR, None, 0, 0, PTR, None) != 0
    assert "e3dgs_distill_forward" in text()
    assert hip_lib.e3dgs_distill_backward(*head, PTR, PTR, PTR, a["row_stride"], a["class_stride"], None) != 0
    assert "e3dgs_distill_backward" in text()


def test_distill_gradient_layout(hip_lib):
    head = (5, 9, 2, PTR, 9, 1, 0, PTR, 2, 1, 0, PTR, 2, 1, 4, 1.0, 1)
    assert hip_lib.e3dgs_distill_backward(*head, PTR, PTR, PTR, 1, 5, None) != 0
    assert "layout" in text()
    assert hip_lib.e3dgs_distill_forward(*head, PTR, PTR, PTR, PTR, 1, 5, PTR, None) != 0
    assert "layout" in text()
    assert hip_lib.e3dgs_distill_forward(*head, PTR, PTR, None, None, 0, 0, PTR, None) != 0
    assert "null pointer" in text()


def test_workspaces_off_their_boundary(hip_lib):
    off = C.c_void_p(4096 + 4)
    assert hip_lib.e3dgs_layer_norm_backward(3, 4, PTR, 4, PTR, 4, 0, PTR, 0, PTR, PTR, PTR, PTR, PTR, off, None) != 0
    assert "16-byte aligned" in text()
    head = (5, 9, 2, PTR, 9, 1, 0, PTR, 2, 1, 0, PTR, 2, 1, 4, 1.0, 1)
    for stats, scratch in ((off, PTR), (PTR, off)):
        assert hip_lib.e3dgs_distill_forward(*head, stats, PTR, PTR, None, 0, 0, scratch, None) != 0
        assert "8-byte aligned" in text()
    assert hip_lib.e3dgs_distill_backward(*head, off, PTR, PTR, 9, 1, None) != 0
    assert "8-byte aligned" in text()


def test_embedding_past_one_launch(hip_lib):
    """A table whose gradient would take more than 2^32 threads to clear (and 2^52 bytes)."""
    rows, dim = (1 << 31) - 2, 1 << 20
    assert hip_lib.e3dgs_embedding_backward(4, rows, dim, PTR, 4, PTR, dim, 1, 1.0, PTR, PTR, None) != 0
    assert "too many values" in text()


@pytest.mark.parametrize("rows, dim, parts", [(1024, 1 << 20, 64), (4096, 40000, 64), (4096, 16385, 64), (7, 40000, 7), (4096, 16384, 1024),
                                              (4096, 48, 1024), (30, 48, 30), (0, 48, 1)])
def test_layer_norm_scratch(hip_lib, rows, dim, parts):
    """Partial sums of both parameters: long rows leave 64 of them, others one to a workgroup."""
    assert hip_lib.e3dgs_layer_norm_backward_scratch_bytes(rows, dim) == parts * 2 * dim * 4 + 256


@pytest.mark.parametrize("temperature", [1e-39, 1e-6, 1e6, 1e25, -1.0])
def test_distill_temperature(hip_lib, temperature):
    """Temperatures whose reciprocal or square is no fp32 number, and the rest of what distill_loss refuses too."""
    head = (5, 9, 2, PTR, 9, 1, 0, PTR, 2, 1, 0, PTR, 2, 1, 4, temperature, 1)
    assert hip_lib.e3dgs_distill_forward(*head, PTR, PTR, PTR, None, 0, 0, PTR, None) != 0
    assert "temperature" in text()
    assert hip_lib.e3dgs_distill_backward(*head, PTR, PTR, PTR, 9, 1, None) != 0
    assert "temperature" in text()


def test_library_without_the_entry_points(hip_lib, monkeypatch):
    """A library of the same version from before they were added is refused by name."""
    import types
    old = types.SimpleNamespace(**{name: (lambda: _lib.ABI_VERSION) for name in _lib.EXPORTED_SYMBOLS if "distill" not in name})
    monkeypatch.setattr(_lib, "_lib", None)
    monkeypatch.setattr(_lib.C, "CDLL", lambda path: old)
    with pytest.raises(_lib.HipLibraryError, match="e3dgs_distill_forward.*rebuild"):
        _lib.lib()
