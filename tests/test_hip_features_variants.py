"""The kernels that embedding, layer_norm and distill_loss take at certain sizes only: planes of 262144 pixels and more, long rows
in many rows, gradients of scores past 128 MiB; and sums that are whole numbers in every order, where a lost or doubled
chunk, round or partial sum changes the result whatever the size."""
import math

import pytest
import torch

from event_3dgs_amd import features, losses
from test_hip_features import DEV, TYPES, check_distill, check_layer_norm, distill_formula, close, half_step, rand

pytestmark = pytest.mark.gpu


def many_labels(n, classes, k, seed=0):
    """k different classes to a row, in equal steps of which k - 1 stay below `classes`; some entries and rows masked."""
    g = torch.Generator().manual_seed(seed + n + 31 * classes + k)
    first, step = (torch.randint(0, classes, (n, 1), generator=g) for _ in range(2))
    step = 1 + step % ((classes - 1) // k)
    index = (first + step * torch.arange(k)) % classes
    index[torch.rand(n, k, generator=g) < 0.1] = -1
    index[torch.rand(n, generator=g) < 0.2] = -1
    return (torch.randn(n, k, generator=g) * 2).to(DEV), index.to(DEV)


# ------------------------------------------------------------------------------------------------ planes, pixel by pixel
PIXELS = [262144, 262145, 262146]        # 4, 1 and 2 (the value) or 1 (the gradient) neighbouring pixels to a lane


def hard_pixels(z, t, index):
    """Duplicates, scores of -infinity and of the type's lowest value, extreme teachers, at places of every kind of a lane's
    pixels; planes (classes, n) and (k, n), changed in place."""
    classes, n, k = z.shape[0], z.shape[1], t.shape[0]
    low, inf = torch.finfo(z.dtype).min, math.inf
    for at in (0, 9, 258, 1031, n // 2, n - 6):
        index[:, at] = 3                                         # one class, listed k times
        z[classes // 2:, at + 1] = -inf                          # switched off, and not listed
        index[:, at + 1] = index[:, at + 1].remainder(classes // 2)
        z[2:, at + 2] = low
        index[:, at + 2] = 1
        z[:, at + 3] = low                                       # equal shares
        t[0, at + 4], index[0, at + 4] = -inf, 0
        t[:, at + 5] = -inf                                      # no label: its scores do not matter
        z[0, at + 5] = float("nan")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", PIXELS)
@pytest.mark.parametrize("k", [1, 4, 5, 8])
def test_distill_pixels(dtype, n, k):
    classes = 13
    t, index = many_labels(n, classes, k)
    t, index = t.t().contiguous().to(dtype), index.int().t().contiguous()
    z = (rand(classes, n) * 2).to(dtype)
    hard_pixels(z, t, index)
    check_distill(z, t, index, 2.0, 0)


@pytest.mark.parametrize("k", [3, 7])
def test_distill_pixels_off_a_boundary(k):
    n, classes = 262144, 11
    t, index = many_labels(n, classes, k)                        # (labels as rows, int64)
    shifted = rand(classes * n + 1)[1:].view(classes, n)
    check_distill(shifted, t.t(), index.t(), 1.0, 0)
    check_distill(rand(classes, n + 3)[:, :n].bfloat16(), t.t(), index.t(), 1.0, 0)              # planes closely packed again
    check_distill(rand(classes, n + 3).bfloat16()[:, 2:n + 2], t.t(), index.t(), 1.0, 0)         # ... and n + 3 apart
    check_distill(rand(classes, n + 2).half()[:, :n], t.t(), index.t(), 1.0, 0)


@pytest.mark.parametrize("n", PIXELS)
@pytest.mark.parametrize("k", [2, 6])
def test_distill_unusable_pixels(n, k):
    """Pixels whose value is NaN or infinite, and that their neighbours are not."""
    classes, inf = 12, math.inf
    t, index = many_labels(n, classes, k)
    t, index = t.t().contiguous(), index.t().contiguous()
    index[0] = 0                                                 # every pixel has a label
    t[0] = 1.0
    z = rand(classes, n) * 2
    broken, nan, off, wanted, teacher = 5, 1026, n // 2 + 3, n - 1, 70001
    index[k - 1, broken] = classes
    z[5, nan] = float("nan")
    z[:, off] = -inf
    index[:, wanted] = 1
    z[1, wanted] = -inf
    t[0, teacher] = float("nan")
    value, d = losses.distill_loss_raw(z, t, index, reduction="none", class_dim=0)
    leaf = z.clone().requires_grad_(True)
    rows = losses.distill_loss(leaf, t, index, reduction="none", class_dim=0)
    (grad,) = torch.autograd.grad(rows, leaf, torch.ones_like(rows))
    assert torch.equal(torch.nan_to_num(value, nan=7.0), torch.nan_to_num(rows, nan=7.0))
    assert torch.equal(torch.nan_to_num(d, nan=7.0), torch.nan_to_num(grad, nan=7.0))
    bad = torch.zeros(n, dtype=torch.bool, device=DEV)
    bad[[broken, nan, off, teacher]] = True
    assert torch.isnan(value[bad]).all() and value[wanted] == inf
    assert torch.isnan(d[:, [broken, nan, off]]).all()
    assert torch.isnan(d[index[:, teacher].clamp(min=0), teacher]).all()
    good = ~bad
    assert torch.isfinite(d[:, good]).all()
    good[wanted] = False
    row, _, _, row_tol, _ = distill_formula(z.t()[good], t.t()[good], index.t()[good], 1.0)
    close(value[good], row, row_tol + 2.0 ** -24 * row.abs(), "the other pixels")


def test_distill_pixels_streamed():
    """Gradients past 128 MiB, four pixels to a lane, long and short lists."""
    n, classes = 700000, 53
    for k, dtype in ((4, torch.float32), (8, torch.float32), (6, torch.bfloat16)):
        wide = classes if dtype == torch.float32 else 101
        t, index = many_labels(n, wide, k)
        check_distill((rand(wide, n) * 2).to(dtype), t.t().contiguous(), index.t().contiguous(), 1.0, 0, reductions=("mean",))


# ------------------------------------------------------------------------------------------------ rows
@pytest.mark.parametrize("dtype, rows, classes", [
    (torch.bfloat16, 20000, 4001), (torch.float32, 9000, 4007), (torch.float16, 9000, 9001), (torch.bfloat16, 4096, 20011),
    (torch.float32, 1100, 40009)])
def test_distill_row_gradients_streamed(dtype, rows, classes):
    """Gradients of a separate backward call past 128 MiB: 64, 256 and 1024 lanes to a row, the listed classes stored again
    behind the streamed ones."""
    stride = (classes + 7) // 8 * 8
    t, index = many_labels(rows, classes, 6)
    index[3], index[rows - 2] = 7, classes - 1                   # a class listed six times
    index[4], index[rows - 3] = -1, -1
    index[9] = 3
    for z in ((rand(rows, classes) * 2).to(dtype),               # packs between single values, other ones in every row
              (rand(rows, stride) * 2).to(dtype)[:, :classes]):  # scores and gradient do not lie alike: value by value
        z[4] = float("nan")                                      # (not looked at)
        z[9, 100:200] = -math.inf
        check_distill(z, t, index, 2.0, reductions=("mean",))
    even = (rand(rows, stride, seed=1) * 2).to(dtype)            # every row on a 16-byte boundary
    t, index = many_labels(rows, stride - 1, 6)
    index[3], index[rows - 2], index[4] = 7, stride - 1, -1
    check_distill(even, t, index, 2.0, reductions=("sum",))
    index[5, 1] = stride                                         # a broken row makes its own gradient NaN
    leaf = even.requires_grad_(True)
    (d,) = torch.autograd.grad(losses.distill_loss(leaf, t, index, 2.0, "none").sum(), leaf)
    bad = (index >= stride).any(1)
    assert torch.isnan(d[bad]).all() and torch.isfinite(d[~bad]).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [8196, 12290, 12292, 16380, 16382, 16384])
def test_layer_norm_long_rows_in_many_rows(dtype, dim):
    """From 1024 rows on the gradient keeps up to 16384 values of a row in registers."""
    for n in (1024, 1100):
        check_layer_norm((rand(n, dim) + 0.5).to(dtype), (1 + 0.2 * rand(dim)).to(dtype), rand(dim, seed=3).to(dtype),
                         rand(n, dim, seed=4).to(dtype))


# ------------------------------------------------------------------------------------------------ sums that are exact
def whole(*shape, seed=0, most=4, dtype=torch.float32):
    g = torch.Generator(device=DEV).manual_seed(seed + sum(shape))
    return torch.randint(-most, most + 1, shape, generator=g, device=DEV).to(dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n, dim", [
    (256, 48), (300, 7), (1024, 66), (1025, 33), (4096, 48), (4097, 5), (16384, 48), (16385, 48), (30011, 257), (131072, 20), (131073, 6),
    (262144, 8), (262145, 3), (1048576, 2), (1048577, 4), (2097152, 1), (2097153, 3)])
def test_embedding_gradient_of_whole_numbers(dtype, n, dim):
    """One row for all positions, two, and many: every partial sum is a whole number of at most 4 n < 2^24, so the sum is
    exact in every order, and the result is the exact one rounded once."""
    d = whole(n, dim, dtype=dtype)
    flat = d.double()
    for rows, how in ((1, None), (2, None), (300, 4.0), (5000, 1.0)):
        g = torch.Generator(device=DEV).manual_seed(n + rows)
        index = (torch.rand(n, generator=g, device=DEV).double().pow(how or 1.0) * rows).long().clamp_(max=rows - 1)
        if rows > 2:
            index[torch.rand(n, generator=g, device=DEV) < 0.1] = -1
        table = torch.zeros(rows, dim, dtype=dtype, device=DEV, requires_grad=True)
        (got,) = torch.autograd.grad(features.embedding(index, table, 0.5), table, d)
        there = index >= 0
        if rows <= 2:
            want = torch.stack([flat[index == r].sum(0) for r in range(rows)]) * 0.5
        else:
            want = torch.zeros(rows, dim, dtype=torch.float64, device=DEV).index_add_(0, index[there], flat[there]) * 0.5
        assert torch.equal(got, want.to(dtype)), rows


def exact_rows(n, dim, seed=0):
    """Rows of small whole numbers with mean 0 and variance 4 in every order of summation: the normalised values are halves of
    whole numbers.  Pairs of 2 and -2, and behind them 3, -3, 1, -1, 0 (sum 0, squares 20 of 5 values) where dim is odd."""
    row = torch.tensor([2.0, -2.0] * (dim // 2 if dim % 2 == 0 else (dim - 5) // 2) + ([] if dim % 2 == 0 else [3.0, -3.0, 1.0, -1.0, 0.0]))
    g = torch.Generator().manual_seed(seed + n + dim)
    orders = torch.stack([torch.randperm(dim, generator=g) for _ in range(min(n, 31))])
    return row[orders][torch.arange(n) % len(orders)].to(DEV) * (1 - 2 * (torch.arange(n) // 7 % 2)).unsqueeze(1).to(DEV)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n, dim", [
    (3, 48), (301, 48), (20000, 48), (100003, 48), (5003, 59), (200000, 59), (9001, 5), (30112, 483), (20000, 300), (3000, 264),
    (1300, 257), (8192, 1024), (2000, 1446), (5000, 514), (4000, 2052), (2000, 4097), (4096, 4096), (3001, 8192), (70, 8193), (1100, 12290),
    (1100, 16384), (70, 16392), (300, 40001), (2100, 20000)])
def test_layer_norm_sums_of_whole_numbers(dtype, n, dim):
    """The parameters' gradients of such rows: sums of halves below 2^24, exact in every order."""
    x = exact_rows(n, dim).to(dtype).requires_grad_(True)
    w, b = (torch.ones(dim, device=DEV, requires_grad=True) for _ in range(2))
    d = whole(n, dim, dtype=dtype)
    y = features.layer_norm(x, w, b, 0.0)
    h = x.detach().double() / 2
    assert torch.equal(y.detach(), (h + 1).to(dtype))
    dx, dw, db = torch.autograd.grad(y, (x, w, b), d)
    g = d.double()
    assert torch.equal(dw.double(), (g * h).sum(0)) and torch.equal(db.double(), g.sum(0))
    ref = (g - g.mean(1, keepdim=True) - h * (g * h).mean(1, keepdim=True)) / 2
    # the sums are exact, the means and dx take six roundings of values of at most |g| + |mean g| + |h mean(g h)|
    mag = (g.abs() + g.mean(1, keepdim=True).abs() + (h * (g * h).mean(1, keepdim=True)).abs()) / 2
    close(dx, ref, half_step(ref, dtype) * 1.01 + 6 * 2.0 ** -24 * mag, "dx")
