"""embedding, layer_norm and distill_loss on the GPU against their formulas in 64 bits.

u = 2^-24 is the rounding of one fp32 operation, a result of type t is off by finfo(t).eps / 2 relative to its value.  A sum
of m terms formed in a tree whose longest path has d additions is off by at most d u times the sum of the absolute terms."""
import math

import pytest
import torch

from event_3dgs_amd import features, losses

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
TYPES = [torch.float32, torch.float16, torch.bfloat16]
DEV = "cuda"


def half_step(ref, dtype):
    """Half a step of `dtype` at ref, the spacing of its subnormals included."""
    f = torch.finfo(dtype)
    return ref.abs() * (f.eps / 2) + f.tiny * f.eps / 2


def close(got, ref, tol, what=""):
    got, ref = got.double(), ref.double()
    assert got.shape == ref.shape, what
    over = ((got - ref).abs() - tol).max().item() if got.numel() else -1.0
    assert torch.isfinite(got).all(), what
    assert over <= 0, "%s: off by %.3g more than allowed" % (what, over)


def rand(*shape, seed=0, scale=1.0):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed + 7919 * len(shape) + sum(shape))).to(DEV) * scale


def tokens(n, rows, seed=0, skew=1.0, empty=0.0):
    g = torch.Generator().manual_seed(seed + n + rows)
    i = (torch.rand(n, generator=g).double().pow(skew) * rows).long().clamp_(max=rows - 1)
    if empty:
        i[torch.rand(n, generator=g) < empty] = -1
    return i.to(DEV)


# ------------------------------------------------------------------------------------------------ embedding
def check_embedding(index, table, scale, d_out):
    leaf = table.detach().requires_grad_(True)
    out = features.embedding(index, leaf, scale)
    dt, flat = table.dtype, index.reshape(-1).long()
    there = (flat >= 0) & (flat < table.shape[0])
    want = torch.zeros(flat.numel(), table.shape[1], dtype=torch.float32, device=DEV)
    want[there] = table.detach().float()[flat[there]] * scale
    want[flat >= table.shape[0]] = float("nan")
    want = want.to(dt).reshape(out.shape)                       # (one fp32 product, rounded once: the same bits)
    assert torch.equal(torch.nan_to_num(out, nan=7.0), torch.nan_to_num(want, nan=7.0))
    out.backward(d_out)
    d = d_out.double().reshape(-1, table.shape[1])[there]
    zero = lambda: torch.zeros(table.shape, dtype=torch.float64, device=DEV)      # noqa: E731
    ref = zero().index_add_(0, flat[there], d) * scale
    mag = zero().index_add_(0, flat[there], d.abs()) * abs(scale)
    count = torch.bincount(flat[there], minlength=table.shape[0]).double().unsqueeze(1)
    close(leaf.grad, ref, half_step(ref, dt) * 1.01 + (count + 2) * U * mag, "embedding gradient")
    assert leaf.grad.dtype == dt
    assert (leaf.grad[(count == 0).squeeze(1)] == 0).all()
    return leaf.grad


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n, rows, dim, skew", [
    (1, 1, 1, 1), (1, 50, 64, 1), (2, 1, 3, 1), (63, 7, 5, 1), (64, 9, 8, 1), (65, 300, 48, 1), (513, 3, 17, 1),
    (1000, 1000, 33, 4), (4097, 70000, 4, 1), (5000, 129, 130, 2), (777, 65, 1000, 2), (20000, 40, 48, 4), (3001, 5, 520, 1)])
def test_embedding(dtype, n, rows, dim, skew):
    check_embedding(tokens(n, rows, skew=skew, empty=0.1), rand(rows, dim).to(dtype), 1.75, rand(n, dim, seed=1).to(dtype))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [2, 6, 12, 20, 66, 132, 1186])
@pytest.mark.parametrize("n, rows", [(130, 1), (256, 9), (255, 3001), (257, 2), (2900, 5)])
def test_embedding_rows_of_four_and_eight_bytes(dtype, dim, n, rows):
    check_embedding(tokens(n, rows, skew=2, empty=0.05), rand(rows, dim).to(dtype), 1.0, rand(n, dim, seed=1).to(dtype))


@pytest.mark.parametrize("rows, dim", [(1, 48), (1, 1), (257, 256), (1, 2052)])
def test_embedding_one_row_for_all(rows, dim):
    n = 30011
    check_embedding(torch.full((n,), rows - 1, dtype=torch.int32, device=DEV), rand(rows, dim), 0.5, rand(n, dim, seed=2))


def test_embedding_orders_and_shapes():
    index = tokens(600, 50).reshape(20, 30)
    table = rand(50, 24)
    a = check_embedding(index.t(), table, 1.0, rand(30, 20, 24))                      # a transposed index
    big = rand(50, 2, 24)
    check_embedding(index.int(), big[:, 1], 1.0, rand(20, 30, 24))                    # table rows 48 apart
    check_embedding(index, rand(24, 50).t(), 1.0, rand(20, 30, 24))                   # a transposed table
    check_embedding(index, rand(50 * 24 + 1)[1:].view(50, 24), 2.0, rand(20, 30, 24))  # off a 16-byte boundary
    check_embedding(index, table, 1.0, rand(20, 24, 30).transpose(1, 2))              # a gradient in another order
    check_embedding(index, table, 1.0, rand(1, 1, 24).expand(20, 30, 24))             # one gradient row for all
    check_embedding(index, table, 1.0, rand(1).expand(20, 30, 24))                    # one value for all
    assert torch.equal(a, check_embedding(index.t(), table, 1.0, rand(30, 20, 24)))   # the same bits again
    out = features.embedding(torch.tensor(3, device=DEV), table)
    assert out.shape == (24,) and torch.equal(out, table[3])


def test_embedding_nothing_to_look_up():
    for index in (torch.empty(0, dtype=torch.int64, device=DEV), torch.full((70,), -1, device=DEV)):
        check_embedding(index, rand(5, 12), 1.0, rand(index.numel(), 12))
    check_embedding(torch.empty(0, 3, dtype=torch.int32, device=DEV), rand(4, 3).half(), 1.0, rand(0, 3, 3).half())
    for dim in (8, 7, 2, 1):
        for dtype in TYPES:
            none = torch.empty(0, dim, device=DEV, dtype=dtype)
            assert (features.embedding(torch.full((2,), -5, device=DEV), none) == 0).all()
            assert torch.isnan(features.embedding(torch.zeros(2, dtype=torch.int64, device=DEV), none)).all()


def test_embedding_index_past_the_table():
    index = torch.tensor([0, 5, 2 ** 40, -2 ** 40, 4, 4], device=DEV)
    check_embedding(index, rand(5, 16), 1.0, rand(6, 16))
    check_embedding(torch.tensor([2 ** 31 - 1, 4, -2 ** 31], dtype=torch.int32, device=DEV), rand(5, 3), 1.0, rand(3, 3))


def test_embedding_special_values():
    table = torch.tensor([[float("inf"), 1.0], [float("nan"), 2.0], [6e4, 3.0]], device=DEV, dtype=torch.float16)
    out = features.embedding(torch.tensor([0, 1, 2, -1], device=DEV), table, 2.0)
    assert torch.isinf(out[0, 0]) and torch.isnan(out[1, 0]) and torch.isinf(out[2, 0]) and (out[3] == 0).all()


def test_embedding_past_32_bits():
    rows, dim = 70000, 32768                                     # 2.3 G values of the table, 4.6 GB
    table = torch.zeros(rows, dim, dtype=torch.bfloat16, device=DEV)
    table[-1] = 3.0
    table[rows - 2] = 5.0
    leaf = table.requires_grad_(True)
    out = features.embedding(torch.tensor([rows - 1, 0, rows - 2, rows - 1], device=DEV), leaf)
    assert (out[0] == 3).all() and (out[1] == 0).all() and (out[2] == 5).all()
    (g,) = torch.autograd.grad(out, leaf, torch.ones_like(out))
    assert (g[-1] == 2).all() and (g[-2] == 1).all() and (g[0] == 1).all() and g[1:-2].count_nonzero() == 0
    del out, g, leaf, table
    n = 2_200_000                                                # 2.25 G values of the output
    small = rand(7, 1024).half()
    index = tokens(n, 7)
    out = features.embedding(index, small)
    assert torch.equal(out[-1000:], small[index[-1000:]]) and torch.equal(out[n // 2:n // 2 + 1000], small[index[n // 2:n // 2 + 1000]])


# ------------------------------------------------------------------------------------------------ layer norm
def check_layer_norm(x, w, b, d_out, eps=1e-5):
    dt = x.dtype
    leaves = [t.detach().requires_grad_(True) if t is not None else None for t in (x, w, b)]
    out = features.layer_norm(*leaves, eps)
    assert out.dtype == dt and out.shape == x.shape
    X = x.detach().double().reshape(-1, x.shape[-1])
    G = d_out.double().reshape(X.shape)
    W = torch.ones(X.shape[1], dtype=torch.float64, device=DEV) if w is None else w.detach().double()
    B = torch.zeros(X.shape[1], dtype=torch.float64, device=DEV) if b is None else b.detach().double()
    mean = X.mean(1, keepdim=True)
    rstd = (X.sub(mean).square().mean(1, keepdim=True) + eps).rsqrt()
    h = (X - mean) * rstd
    # 256 u: a path of fewer than 128 additions for the mean and for the variance, and the products behind them
    eh = 256 * U * ((X.abs().mean(1, keepdim=True) + X.abs()) * rstd + h.abs())
    ref = h * W + B
    close(out.reshape(X.shape), ref, half_step(ref, dt) * 1.01 + eh * W.abs() + 2 * U * ref.abs(), "layer norm")
    out.backward(d_out)
    g = G * W
    s1, s2 = g.mean(1, keepdim=True), (g * h).mean(1, keepdim=True)
    dx = rstd * (g - s1 - h * s2)
    gm, ghm = g.abs().mean(1, keepdim=True), (g * h).abs().mean(1, keepdim=True)
    tol = rstd * (256 * U * (g.abs() + gm + h.abs() * ghm) + eh * ghm + h.abs() * (g.abs() * eh).mean(1, keepdim=True))
    tol = tol + 256 * U * dx.abs()                                   # rstd itself
    close(leaves[0].grad.reshape(X.shape), dx, half_step(dx, dt) * 1.01 + tol, "dx")
    n = X.shape[0]
    if w is not None:
        ref = (G * h).sum(0)
        close(leaves[1].grad, ref, half_step(ref, w.dtype) * 1.01 + (G.abs() * eh).sum(0) + (n + 4) * U * (G * h).abs().sum(0), "dw")
    if b is not None:
        ref = G.sum(0)
        close(leaves[2].grad, ref, half_step(ref, b.dtype) * 1.01 + (n + 4) * U * G.abs().sum(0), "db")
    return [t.grad for t in leaves if t is not None]


DIMS = [1, 2, 3, 8, 17, 32, 48, 59, 63, 64, 65, 128, 200, 256, 257, 512, 520, 1000, 1024, 1032, 2048, 2056, 4096, 4100, 8192]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", DIMS)
def test_layer_norm(dtype, dim):
    n = 37 if dim > 64 else 301
    check_layer_norm((rand(n, dim) * 2 + 0.5).to(dtype), (1 + 0.2 * rand(dim)).to(dtype), rand(dim, seed=3).to(dtype),
                     rand(n, dim, seed=4).to(dtype))


@pytest.mark.parametrize("dtype, dim", [(torch.float32, 4104), (torch.float32, 10001), (torch.bfloat16, 16392), (torch.float16, 9001),
                                        (torch.bfloat16, 40000)])
def test_layer_norm_long_rows(dtype, dim):
    for n in (1, 70):
        check_layer_norm(rand(n, dim).to(dtype), rand(dim, seed=1).to(dtype), rand(dim, seed=2).to(dtype), rand(n, dim, seed=3).to(dtype))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [514, 516, 1020, 1026, 1446, 1537, 2050, 2052, 4090, 4097, 4100, 4588, 8190, 8193, 8196, 8200, 12290,
                                 16382, 16384, 16386, 16388, 16392])
def test_layer_norm_rows_of_four_and_eight_bytes(dtype, dim):
    """Long rows on boundaries of 2, 4, 8 and 16 bytes, up to where another kernel takes over; one workgroup and several."""
    for n in (3, 11):
        check_layer_norm((rand(n, dim) + 0.5).to(dtype), (1 + 0.2 * rand(dim)).to(dtype), rand(dim, seed=3).to(dtype),
                         rand(n, dim, seed=4).to(dtype))


@pytest.mark.parametrize("n, dim", [(0, 8), (1, 48), (2, 4096), (20000, 48), (9000, 5), (5003, 59), (3000, 264)])
def test_layer_norm_row_counts(n, dim):
    grads = check_layer_norm(rand(n, dim), rand(dim), rand(dim, seed=1), rand(n, dim, seed=2))
    again = check_layer_norm(rand(n, dim), rand(dim), rand(dim, seed=1), rand(n, dim, seed=2))
    assert all(torch.equal(a, b) for a, b in zip(grads, again))
    if n == 0:
        assert (grads[1] == 0).all() and (grads[2] == 0).all()


def test_layer_norm_parameters_and_orders():
    x, d = rand(40, 96), rand(40, 96, seed=1)
    check_layer_norm(x, None, None, d)
    check_layer_norm(x, rand(96), None, d)
    check_layer_norm(x, None, rand(96), d)
    check_layer_norm(x.half(), rand(96), rand(96, seed=5), d.half())                     # fp32 parameters of fp16 rows
    check_layer_norm(x, rand(96).bfloat16(), rand(96, seed=5).bfloat16(), d)
    check_layer_norm(rand(40, 2, 96)[:, 1], rand(96), rand(96, seed=5), d)               # rows 192 apart
    check_layer_norm(rand(96, 40).t(), rand(96), rand(96, seed=5), rand(96, 40, seed=2).t())
    check_layer_norm(rand(40 * 96 + 1)[1:].view(40, 96), rand(96), rand(96, seed=5), d)   # off a 16-byte boundary
    check_layer_norm(rand(4, 10, 96), rand(192)[::2], rand(96, seed=5), rand(96).expand(4, 10, 96))
    check_layer_norm(rand(96), rand(96, seed=4), rand(96, seed=5), rand(96, seed=6))     # a single row without a batch
    # a part of the gradients
    xl, wl = x.detach().requires_grad_(True), rand(96).requires_grad_(True)
    full = torch.autograd.grad(features.layer_norm(xl, wl), (xl, wl), d)
    assert torch.equal(torch.autograd.grad(features.layer_norm(xl, wl.detach()), xl, d)[0], full[0])
    assert torch.equal(torch.autograd.grad(features.layer_norm(x, wl), wl, d)[0], full[1])


def test_layer_norm_hard_rows():
    check_layer_norm(torch.full((3, 50), 4.0, device=DEV), rand(50), rand(50, seed=1), rand(3, 50))      # no variance
    check_layer_norm(rand(5, 200) + 1000.0, rand(200), rand(200, seed=1), rand(5, 200))                # far from zero
    check_layer_norm(rand(5, 200) * 1e-4, rand(200), rand(200, seed=1), rand(5, 200))
    check_layer_norm(rand(5, 1), rand(1), rand(1, seed=1), rand(5, 1))
    x = rand(4, 64)
    x[1, 3], x[2, 5] = float("nan"), float("inf")
    out = features.layer_norm(x)
    assert torch.isnan(out[1]).all() and torch.isnan(out[2]).all() and torch.isfinite(out[[0, 3]]).all()


def test_layer_norm_past_32_bits():
    n, dim = 1_100_000, 2048                                     # 2.25 G values
    x = torch.zeros(n, dim, dtype=torch.bfloat16, device=DEV)
    x[-3:] = rand(3, dim).bfloat16()
    x[n // 2] = rand(dim, seed=1).bfloat16()
    leaf = x.requires_grad_(True)
    out = features.layer_norm(leaf)
    for row in (n // 2, n - 2, n - 1):
        assert torch.equal(out[row], features.layer_norm(x.detach()[row]))
    d = torch.zeros_like(x)
    d[-1] = rand(dim, seed=2).bfloat16()
    (dx,) = torch.autograd.grad(out, leaf, d)
    one = x.detach()[-1:].requires_grad_(True)
    (want,) = torch.autograd.grad(features.layer_norm(one), one, d[-1:])
    assert torch.equal(dx[-1], want[0]) and dx[:10].count_nonzero() == 0


# ------------------------------------------------------------------------------------------------ distillation
def label(n, classes, k, seed=0, empty=0.2):
    g = torch.Generator().manual_seed(seed + n + 31 * classes + k)
    index = torch.stack([torch.randperm(classes, generator=g)[:k] for _ in range(n)]) if n else torch.zeros(0, k, dtype=torch.int64)
    score = torch.randn(n, k, generator=g) * 2
    if empty and n > 2:
        index[torch.rand(n, k, generator=g) < 0.1] = -1
        index[torch.rand(n, generator=g) < empty] = -1
    return score.to(DEV), index.to(DEV)


def distill_formula(z, t, index, temp):
    """Per row in 64 bits: value, gradient, labelled, and the bounds of both (classes last)."""
    z, t, index = z.double(), t.double(), index.long()
    there = (index >= 0) & (t > -math.inf)
    any_ = there.any(1)
    z = torch.where(any_.unsqueeze(1), z, 0.0)                   # (a row without a label does not look at its scores)
    top = torch.where(there, t, -math.inf).amax(1, keepdim=True)
    top = torch.where(any_.unsqueeze(1), top, 0.0)
    w = torch.where(there, ((t - top) / temp).exp(), 0.0)
    q = torch.where(any_.unsqueeze(1), w / w.sum(1, keepdim=True).clamp_min(1e-300), 0.0)
    m = z.amax(1, keepdim=True)
    s = ((z - m) / temp).exp().sum(1, keepdim=True)
    at = index.clamp(min=0)
    logq = (t - top) / temp - w.sum(1, keepdim=True).clamp_min(1e-300).log()
    zm = z.gather(1, at) - m
    used = q > 0
    row = temp ** 2 * torch.where(used, q * (logq - (zm / temp - s.log())), 0.0).sum(1)
    p = ((z - m) / temp).exp() / s
    Q = torch.zeros_like(z).scatter_add_(1, at, q)
    grad = torch.where(any_.unsqueeze(1), temp * (p - Q), 0.0)
    # exponent (z - m) / T times log2 e: 4 roundings of the exponent (times ln 2 < 1), one of exp2 and one of the product; the
    # sums (a path of fewer than 256 additions) and their reciprocals
    far = torch.where(p > 0, (z - m).abs() / temp, 0.0)
    sums = 300 * U + (p * 8 * U * far).sum(1, keepdim=True)
    qfar = torch.where(used, (t - top).abs() / temp, 0.0)
    qsums = 300 * U + (q * 8 * U * qfar).sum(1, keepdim=True)
    eq = q * (8 * U * qfar + qsums)
    tol = temp * (p * (8 * U * far + sums) + torch.zeros_like(z).scatter_add_(1, at, eq)) + 2e-38
    parts = torch.where(used, q * (logq.abs() + zm.abs() / temp + s.log().abs() + 1), 0.0).sum(1)
    qlog = torch.where(used, eq * (logq - (zm / temp - s.log())).abs(), 0.0).sum(1)
    row_tol = temp ** 2 * (64 * U * parts + qlog + (sums + qsums).squeeze(1) * any_)
    return row, grad, any_, row_tol, tol


def check_distill(z, t, index, temp=1.0, class_dim=-1, reductions=("none", "mean", "sum"), g=1.5):
    last = lambda v: v.movedim(class_dim, -1).reshape(-1, v.shape[class_dim])       # noqa: E731
    row, grad, any_, row_tol, tol = distill_formula(last(z.detach()), last(t), last(index), temp)
    n = max(1, int(any_.sum()))
    for how in reductions:
        leaf = z.detach().requires_grad_(True)
        value = losses.distill_loss(leaf, t, index, temp, how, class_dim)
        raw, d_raw = losses.distill_loss_raw(leaf, t, index, temp, how, class_dim)
        assert value.dtype == raw.dtype == torch.float32 and not d_raw.requires_grad
        weight = 1.0 / n if how == "mean" else 1.0
        if how == "none":
            for v in (value, raw):
                close(v.reshape(-1), row, row_tol + U * row.abs(), "rows")
            up = rand(*value.shape, seed=9) if value.dim() else torch.tensor(g, device=DEV)
            by_row = up.double().reshape(-1, 1)
        else:
            for v in (value, raw):
                close(v, row.sum() * weight, (row_tol.sum() + 20 * U * row.abs().sum()) * weight + U * abs(row.sum()) * weight, how)
            up, by_row = torch.tensor(g, device=DEV), g
        value.backward(up)
        for got, f in ((leaf.grad, by_row), (d_raw, 1.0)):
            assert got.dtype == z.dtype and got.shape == z.shape
            ref = grad * weight * f
            scale = abs(f) if isinstance(f, float) else f.abs()
            close(last(got), ref, half_step(ref, z.dtype) * 1.01 + (tol + 4 * U * grad.abs()) * weight * scale, how + " gradient")
            assert (last(got)[~any_] == 0).all()
    return leaf.grad


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n, classes, k, temp", [
    (1, 1, 1, 1.0), (3, 2, 1, 1.0), (70, 7, 7, 2.0), (33, 19, 3, 1.0), (17, 64, 5, 0.5), (40, 65, 64, 1.0), (9, 151, 8, 2.0),
    (21, 1000, 20, 1.0), (600, 50, 2, 1.0), (5, 2048, 100, 4.0), (30, 40, 40, 1.0), (2, 9000, 1000, 1.0), (700, 5000, 9, 1.0), (6, 2049, 33, 1.0), (3, 16384, 7, 1.0), (2, 16391, 300, 2.0), (2, 50001, 64, 1.0),
                                                (1100, 2100, 3, 2.0), (1024, 3001, 70, 1.0), (1030, 4001, 2, 1.0), (1050, 8000, 5, 1.0), (1040, 9000, 3, 1.0),
                                                (300, 20000, 3, 1.0)])
def test_distill_rows(dtype, n, classes, k, temp):
    t, index = label(n, classes, k)
    check_distill((rand(n, classes) * 3).to(dtype), t.to(dtype), index.int(), temp)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("classes, h, w, k", [(2, 5, 3, 1), (3, 9, 17, 3), (8, 8, 8, 4), (64, 13, 31, 4), (40, 4, 8, 7), (9, 2, 32, 8), (20, 6, 6, 9), (151, 7, 10, 20), (256, 6, 11, 2), (300, 5, 6, 3)])
def test_distill_planes(dtype, classes, h, w, k):
    t, index = label(h * w, classes, k)
    t, index = (v.t().reshape(k, h, w) for v in (t, index))
    check_distill((rand(classes, h, w) * 3).to(dtype), t.contiguous(), index.contiguous(), 2.0, 0)


def test_distill_many_rows():
    t, index = label(700, 33, 3)
    t, index = t.repeat(30, 1), index.repeat(30, 1)              # 21000 rows: more than one round of every workgroup
    z = rand(21000, 33) * 2
    a = check_distill(z, t, index)
    assert torch.equal(a, check_distill(z, t, index))
    many = 300000                                                # more pixels than one round of the plane layout
    t, index = t.repeat(15, 1)[:many], index.repeat(15, 1)[:many]
    check_distill(rand(33, many) * 2, t.t(), index.t(), class_dim=0, reductions=("mean",))


def test_distill_value_of_long_lists():
    """A list of every class, each twice: q and p differ by the scores alone."""
    for classes in (100, 512):
        index = torch.arange(classes, device=DEV).repeat(1, 2).expand(3, -1)
        check_distill(rand(3, classes) * 2, rand(3, 2 * classes), index, 2.0)
        if classes == 100:
            check_distill((rand(3, classes) * 2).t().contiguous(), rand(3, 2 * classes).t(), index.t(), 2.0, 0)


def test_distill_layouts():
    t, index = label(24, 40, 5)
    z = rand(24, 40)
    want = check_distill(z, t, index)
    assert torch.equal(check_distill(z.clone(), t.clone(), index.clone()), want)
    check_distill(rand(24, 100)[:, 30:70], t, index)                                         # rows 100 apart, off a boundary
    check_distill(rand(24 * 40 + 1)[1:].view(24, 40), t, index)
    check_distill(z.reshape(4, 6, 40), t.reshape(4, 6, 5), index.reshape(4, 6, 5))
    check_distill(z.reshape(4, 6, 40).transpose(0, 1), t.reshape(4, 6, 5).transpose(0, 1), index.reshape(4, 6, 5).transpose(0, 1))
    check_distill(z.reshape(2, 12, 40).transpose(1, 2), t.reshape(2, 12, 5).transpose(1, 2), index.reshape(2, 12, 5).transpose(1, 2), class_dim=1)
    check_distill(z, t[:, :1].expand(24, 5), index)                                          # one score for all entries
    check_distill(z[0], t[0], index[0].clamp(min=0))                                         # a single row without a batch
    check_distill(z.bfloat16(), t.half(), index.int())
    empty = torch.empty(0, 9, device=DEV)
    value, d = losses.distill_loss_raw(empty, empty[:, :2], torch.empty(0, 2, dtype=torch.int32, device=DEV))
    assert value.item() == 0 and d.shape == (0, 9)


@pytest.mark.parametrize("planes", [False, True])
@pytest.mark.parametrize("classes", [12, 200, 5000])
def test_distill_labels(planes, classes):
    """Rows without a label, masked entries, the same class twice, unusable logits in rows that do not count."""
    inf = math.inf
    z = rand(8, classes) * 2
    t = torch.tensor([[1.0, 2.0, 0.5], [1.0, -inf, 3.0], [-inf, -inf, -inf], [0.0, 0.0, 0.0], [1.0, 1.0, 2.0], [5.0, 1.0, 1.0],
                      [1e4, -1e4, 0.0], [2.0, float("nan"), 1.0]], device=DEV)
    index = torch.tensor([[3, 3, 3], [1, 2, 4], [1, 2, 3], [-1, -1, -1], [5, 7, 5], [0, -1, classes - 1], [1, 2, 3], [4, -1, 6]], device=DEV)
    z[2, 1], z[3] = float("nan"), inf                            # rows 2 and 3 have no label
    z[0, 7:10], z[1, 8] = -inf, torch.finfo(torch.float32).min   # classes that are switched off
    if planes:
        check_distill(z.t().contiguous(), t.t(), index.t(), class_dim=0)
    else:
        check_distill(z, t, index)
    # no label at all
    value, d = losses.distill_loss_raw(z, t, torch.full_like(index, -1))
    assert value.item() == 0 and (d == 0).all()


@pytest.mark.parametrize("planes", [False, True])
@pytest.mark.parametrize("classes", [12, 200, 5000])
def test_distill_unusable_rows(planes, classes):
    inf = math.inf
    z = rand(6, classes)
    t = torch.ones(6, 2, device=DEV)
    index = torch.tensor([[1, 2], [1, classes], [1, 2], [1, 2], [1, 2], [1, 2]], device=DEV)
    z[2] = -inf                                                  # every class switched off
    z[3, 5] = float("nan")
    z[4, 1] = -inf                                               # the teacher wants a class that is switched off
    t[5, 0] = float("nan")
    args = (z.t().contiguous(), t.t(), index.t()) if planes else (z, t, index)
    value, d = losses.distill_loss_raw(*args, reduction="none", class_dim=0 if planes else -1)
    d = d.t() if planes else d
    assert torch.isfinite(value[0]) and torch.isfinite(d[0]).all()
    assert torch.isnan(value[[1, 2, 3, 5]]).all() and value[4] == inf
    assert torch.isnan(d[[1, 2, 3]]).all() and torch.isnan(d[5, 1]) and torch.isnan(d[5, 2])
    ref = torch.softmax(z[4], 0)
    ref[1:3] -= 0.5
    close(d[4], ref, 300 * U * (ref.abs() + 1), "a class that is switched off")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows, classes", [(1600, 2500), (1600, 4000), (1600, 5000), (1600, 30), (400, 2500), (300, 17000)])
def test_distill_hard_rows_among_many(dtype, rows, classes):
    """Rows without a label, of one listed class, of switched off classes and of NaN, as many as take another kernel."""
    inf = math.inf
    z = (rand(rows, classes) * 2).to(dtype)
    t, index = label(rows, classes, 4, empty=0.3)
    z[0::7, 1] = -inf
    z[3::11, 2:classes // 2] = torch.finfo(dtype).min
    z[(index < 0).all(1)] = float("nan")                         # not looked at
    z.scatter_(1, index.clamp(min=0), torch.where((index < 0).all(1, keepdim=True), float("nan"), 1.5).to(dtype).expand(-1, 4).contiguous())
    check_distill(z, t, index, 2.0)
    index[5] = classes                                           # a broken row makes its own value and gradient NaN
    value, d = losses.distill_loss_raw(z, t, index, 2.0, "none")
    assert torch.isnan(value[5]) and torch.isnan(d[5]).all()
    assert torch.isfinite(value[6:]).all() and torch.isfinite(d[6:]).all() and torch.isfinite(value[:5]).all()


def test_distill_lowest_values():
    for dtype in TYPES:
        low = torch.finfo(dtype).min
        z = rand(5, 300).to(dtype)
        z[:, 100:] = low
        z[3] = low                                               # all classes at the lowest value: equal shares
        t, index = label(5, 100, 4, empty=0.0)
        for temp in (0.25, 1.0, 4.0):
            check_distill(z, t.to(dtype), index, temp)
            zt = z.t().contiguous()
            check_distill(zt[:200], t.to(dtype).t(), index.t(), temp, class_dim=0)


def test_distill_past_32_bits():
    n, classes = 16500, 131072                                   # 2.16 G scores
    z = torch.zeros(n, classes, dtype=torch.float16, device=DEV)
    z[-1, -1] = 4.0
    t = torch.ones(n, 2, device=DEV)
    index = torch.tensor([0, classes - 1], device=DEV, dtype=torch.int32).expand(n, 2)
    value, d = losses.distill_loss_raw(z, t, index, reduction="none")
    row, grad, _, row_tol, tol = distill_formula(z[-2:], t[-2:], index[-2:], 1.0)
    close(value[-2:], row, row_tol + U * row.abs(), "last rows")
    close(d[-2:], grad, half_step(grad, torch.float16) * 1.01 + tol, "last gradients")


def test_distill_planes_past_32_bits():
    classes, n = 250, 8_650_000                                  # 2.16 G scores
    z = torch.zeros(classes, n, dtype=torch.float16, device=DEV)
    z[:, -4:] = (rand(classes, 4) * 2).half()
    for k in (2, 12):                                            # the label in registers, and in LDS
        t = torch.ones(k, n, device=DEV)
        index = torch.full((k, n), -1, dtype=torch.int32, device=DEV)
        index[:, -4:] = torch.arange(classes - 4 * k, classes, device=DEV, dtype=torch.int32).view(k, 4)
        value, d = losses.distill_loss_raw(z, t, index, reduction="none", class_dim=0)
        row, grad, _, row_tol, tol = distill_formula(z[:, -4:].t(), t[:, -4:].t(), index[:, -4:].t(), 1.0)
        close(value[-4:], row, row_tol + U * row.abs(), "last pixels")
        close(d[:, -4:].t(), grad, half_step(grad, torch.float16) * 1.01 + tol, "last gradients")
        assert (value[:-4] == 0).all() and d[:, :1000].count_nonzero() == 0
        del t, index, value, d


# ------------------------------------------------------------------------------------------------ differences
def test_gradients_against_differences():
    """A step of the inputs along the gradient changes the value by the squared norm of the gradient, to second order.  fp32
    values of size 1 are off by fewer than 1e-5; the step is large enough for that to be 1 % of the difference."""
    table, w, b, head = rand(40, 32), 1 + 0.1 * rand(32), rand(32, seed=1) * 0.1, rand(32, 20, seed=2) * 0.3
    index, (t, ids) = tokens(300, 40), label(300, 20, 4)

    def value(*p):
        return losses.distill_loss(features.layer_norm(features.embedding(index, p[0], 1.5), p[1], p[2]) @ head, t, ids, 1.0)

    for which in range(3):
        p = [x.detach().clone().requires_grad_(i == which) for i, x in enumerate((table, w, b))]
        (g,) = torch.autograd.grad(value(*p), p[which])
        n2 = g.double().square().sum().item()
        h = 0.02 / math.sqrt(n2)
        q = [x.detach() for x in p]
        ends = []
        for sign in (1, -1):
            q[which] = p[which].detach() + sign * h * g
            ends.append(value(*q).item())
        assert abs((ends[0] - ends[1]) / (2 * h) - n2) <= 0.02 * n2 + 1e-5 / h


# ------------------------------------------------------------------------------------------------ streams, graphs, threads
def chain(index, table, w, b, head, t, ids, planes=None):
    rows = features.layer_norm(features.embedding(index, table, 2.0), w, b)
    return losses.distill_loss(rows @ head, t, ids, 2.0)


def chain_inputs(seed=0, n=900):
    t, ids = label(n, 24, 3, seed)
    return dict(index=tokens(n, 60, seed, 2.0, 0.05), table=rand(60, 48, seed=seed), w=1 + 0.1 * rand(48, seed=seed),
                b=rand(48, seed=seed + 1), head=rand(48, 24, seed=seed) * 0.2, t=t, ids=ids)


def chain_grads(v):
    p = {k: x.detach().requires_grad_(k in ("table", "w", "b", "head")) for k, x in v.items()}
    value = chain(**p)
    return [value.detach()] + list(torch.autograd.grad(value, [p[k] for k in ("table", "w", "b", "head")]))


def test_run_together():
    """Lookup, norm, decoder and loss as one training step, against the same step in 64 bits.  Each of the four stages is
    accurate to fewer than 2^-17 of its norm (sums of at most 900 terms in fp32: below 900 u = 2^-14.2 in the worst case of
    the weight sums, which is the bound taken for all)."""
    v = chain_inputs()
    got = chain_grads(v)
    p = {k: (x.double() if x.is_floating_point() else x).detach().requires_grad_(k in ("table", "w", "b", "head")) for k, x in v.items()}
    there = (p["index"] >= 0).unsqueeze(1)
    x = torch.where(there, p["table"][p["index"].clamp(min=0)] * 2.0, 0.0)
    z = torch.nn.functional.layer_norm(x, (48,), p["w"], p["b"]) @ p["head"]
    keep = (p["ids"] >= 0).any(1)
    there, ids = p["ids"][keep] >= 0, p["ids"][keep].clamp(min=0)
    q = torch.softmax(torch.where(there, p["t"][keep] / 2.0, -math.inf), 1)
    logp = torch.log_softmax(z[keep] / 2.0, 1).gather(1, ids)
    value = 4.0 * (torch.xlogy(q, q) - torch.where(there, q * logp, 0.0)).sum() / keep.sum()
    want = [value.detach()] + list(torch.autograd.grad(value, [p[k] for k in ("table", "w", "b", "head")]))
    for a, b in zip(got, want):
        assert (a.double() - b).norm() <= 4 * 2.0 ** -14.2 * b.norm()


def test_run_together_through_the_rasteriser():
    """Codes looked up for every Gaussian, normalised, decoded to three class scores, rendered, and compared per pixel: the
    same step with torch's elementary operations around the same rasteriser gives the same gradients."""
    from event_3dgs_amd import synth
    from event_3dgs_amd.cameras import orbit_camera
    from event_3dgs_amd.renderer import GaussianView, PipelineParams, render
    n, width, height = 4000, 96, 64
    scene = GaussianView(synth.make_scene(n, "trained", seed=0, device=DEV))
    cam = orbit_camera(0, 8, width, height, device=DEV)
    index = tokens(n, 30)
    t, ids = label(height * width, 3, 2)
    t, ids = t.t().reshape(2, height, width), ids.t().reshape(2, height, width)
    v = [rand(30, 16), 1 + 0.1 * rand(16), rand(16, seed=1), rand(16, 3, seed=2)]

    def step(own):
        table, w, b, head = p = [x.detach().clone().requires_grad_(True) for x in v]
        x = features.embedding(index, table) if own else table[index]
        if own:
            x = features.layer_norm(x, w, b)
        else:
            x = x - x.mean(1, keepdim=True)
            x = x / torch.sqrt(x.square().mean(1, keepdim=True) + 1e-5) * w + b
        image = render(cam, scene, PipelineParams(), torch.zeros(3, device=DEV), override_color=x @ head)["render"]
        if own:
            value = losses.distill_loss(image, t, ids, class_dim=0)
        else:
            there, z = ids >= 0, torch.log_softmax(image, 0)
            some = there.any(0)
            q = torch.where(some, torch.softmax(torch.where(there, t, torch.where(some, -math.inf, 0.0)), 0), 0.0)
            rows = torch.where(there, torch.xlogy(q, q) - q * z.gather(0, ids.clamp(min=0)), 0.0).sum(0)
            value = rows.sum() / some.sum()
        return [value.detach()] + list(torch.autograd.grad(value, p))

    # both sides run in fp32: sums of up to 6144 pixels and 4000 Gaussians, 6144 u < 2^-11.4 of the absolute terms
    for a, b in zip(step(True), step(False)):
        assert (a - b).norm() <= 2.0 ** -11.4 * b.norm()


def test_on_another_stream():
    v = chain_inputs(5)
    want = chain_grads(v)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = chain_grads(v)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_captured_and_replayed():
    """Two graphs of the same step on inputs of their own, replayed in turn with eager work between: the eager results."""
    sets = [chain_inputs(k) for k in range(4)]
    want = [chain_grads(v) for v in sets]
    held = [{k: x.clone() for k, x in sets[0].items()} for _ in range(2)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for h in held:
            chain_grads(h)
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for h in held:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(chain_grads(h))
        graphs.append(g)
    for round_ in range(4):
        for i in range(2):
            k = (round_ + 2 * i + 1) % 4
            for name, x in sets[k].items():
                held[i][name].copy_(x)
            graphs[i].replay()
            chain_grads(sets[(k + 1) % 4])
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(outs[i], want[k])), (round_, i)


def test_two_threads():
    import threading
    sets = [chain_inputs(k, 3000) for k in range(2)]
    want = [chain_grads(v) for v in sets]
    torch.cuda.synchronize()
    bad = []

    def work(k):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(10):
                got = chain_grads(sets[k])
                torch.cuda.current_stream().synchronize()
                if not all(torch.equal(a, b) for a, b in zip(got, want[k])):
                    bad.append(k)

    threads = [threading.Thread(target=work, args=(k,)) for k in range(2)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not bad


# ------------------------------------------------------------------------------------------------ refusals
def test_refusals():
    x, i = rand(4, 6), torch.zeros(4, dtype=torch.int64, device=DEV)
    t, ids = rand(4, 2), torch.zeros(4, 2, dtype=torch.int64, device=DEV)
    bad = [
        lambda: features.embedding(i.float(), x), lambda: features.embedding(i, x.double()), lambda: features.embedding(i, x[0]),
        lambda: features.embedding(i.cpu(), x), lambda: features.embedding(i, x, float("inf")),
        lambda: features.embedding(i, x, 1e300), lambda: features.layer_norm(x, eps=1e300),
        lambda: features.layer_norm(x.double()), lambda: features.layer_norm(x, rand(5)), lambda: features.layer_norm(x, rand(6, 1)),
        lambda: features.layer_norm(x, rand(6).cpu()), lambda: features.layer_norm(x, eps=-1.0),
        lambda: features.layer_norm(x, rand(6), rand(6).half()), lambda: features.layer_norm(x[:, :0]),
        lambda: losses.distill_loss(x, t, ids[:, :1]), lambda: losses.distill_loss(x, t[:3], ids[:3]),
        lambda: losses.distill_loss(x, t, ids.float()), lambda: losses.distill_loss(x.double(), t, ids),
        lambda: losses.distill_loss(x, t, ids, temperature=0.0), lambda: losses.distill_loss(x, t, ids, temperature=float("nan")),
        lambda: losses.distill_loss(x, t, ids, class_dim=2), lambda: losses.distill_loss(x, t[:, :0], ids[:, :0]),
        lambda: losses.distill_loss(x, t[0], ids[0]), lambda: losses.distill_loss(x, t.requires_grad_(True), ids),
        lambda: losses.distill_loss(x, rand(4, 1025), torch.zeros(4, 1025, dtype=torch.int32, device=DEV)),
    ]
    for k, call in enumerate(bad):
        with pytest.raises(RuntimeError):
            call()
            pytest.fail("call %d was not refused" % k)


def test_second_derivatives_are_refused():
    x = rand(4, 6).requires_grad_(True)
    t, ids = rand(4, 2), torch.zeros(4, 2, dtype=torch.int64, device=DEV)
    for value in (features.embedding(ids, x).sum(), features.layer_norm(x).square().sum(), losses.distill_loss(x, t, ids)):
        with pytest.raises(RuntimeError, match="once"):
            torch.autograd.grad(value, x, create_graph=True)


def test_inputs_changed_in_between_are_noticed():
    x, t, ids = rand(4, 6).requires_grad_(True), rand(4, 2), torch.zeros(4, 2, dtype=torch.int64, device=DEV)
    value = losses.distill_loss(x, t, ids)
    t += 1
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        value.backward()


@pytest.mark.parametrize("n, rows, dim", [(255, 40, 48), (256, 40, 48), (257, 40, 48), (256, 3, 1000), (1024, 9, 20), (1025, 9, 20),
                                          (4096, 300, 16), (4097, 300, 16), (8192, 20, 12), (8193, 20, 12), (16384, 4000, 8),
                                          (16385, 4000, 8), (300000, 70000, 4), (524288, 255, 3), (524289, 256, 3),
                                          (1048576, 65535, 2), (1048577, 65536, 2), (2097152, 300, 1), (2097153, 300, 1),
                                          (20011, 17000000, 1)])
def test_embedding_sort_sizes(n, rows, dim):
    """Position counts around which another sort takes over, int32 and int64 indices, masked ends."""
    index = tokens(n, rows, skew=2.0, empty=0.2)
    index[-1] = -1
    a = check_embedding(index, rand(rows, dim), 1.0, rand(n, dim, seed=1))
    assert torch.equal(a, check_embedding(index.int(), rand(rows, dim), 1.0, rand(n, dim, seed=1)))
    first = torch.full((n,), rows, device=DEV)                   # all outside the table but one
    first[n // 2] = rows - 1
    check_embedding(first, rand(rows, dim), 1.0, rand(n, dim, seed=2))


@pytest.mark.parametrize("n", [1, 3, 4, 5, 16, 17, 64, 65, 128, 129, 1024, 1025, 1300])
@pytest.mark.parametrize("dim", [1, 7, 16, 64, 100, 300])
def test_layer_norm_few_rows(n, dim):
    """Row counts around which the column sums go from one workgroup to several."""
    check_layer_norm(rand(n, dim) + 0.3, rand(dim), rand(dim, seed=1), rand(n, dim, seed=2))


def test_large_results_are_streamed():
    """Results past 128 MiB are stored past the cache: the same values."""
    n, dim = 900000, 48
    index, table = tokens(n, 500), rand(500, dim)
    leaf = table.clone().requires_grad_(True)
    out = features.embedding(index, leaf, 3.0)
    assert torch.equal(out, table[index] * 3.0)
    out = out.detach().requires_grad_(True)
    y = features.layer_norm(out)
    part = features.layer_norm(out.detach()[-5000:])
    assert torch.equal(y[-5000:], part)
    d = rand(n, dim)
    (dx,) = torch.autograd.grad(y, out, d)
    small = out.detach()[-5000:].requires_grad_(True)
    (want,) = torch.autograd.grad(features.layer_norm(small), small, d[-5000:])
    assert torch.equal(dx[-5000:], want)
    big = rand(700000, 64).requires_grad_(True)                  # a gradient table of 179 MB, most of it empty
    (g,) = torch.autograd.grad(features.embedding(index[:5000], big), big, rand(5000, 64))
    keep = torch.zeros(500, 64, dtype=torch.float64, device=DEV).index_add_(0, index[:5000], rand(5000, 64).double())
    count = torch.bincount(index[:5000], minlength=500).double().unsqueeze(1)
    mag = torch.zeros(500, 64, dtype=torch.float64, device=DEV).index_add_(0, index[:5000], rand(5000, 64).double().abs())
    close(g[:500], keep, half_step(keep, torch.float32) * 1.01 + (count + 2) * U * mag)
    assert g[500:].count_nonzero() == 0


@pytest.mark.parametrize("classes, k", [(300, 3), (40, 257), (300, 1024)])
def test_distill_planes_past_their_limits(classes, k):
    """More than 256 classes or entries in planes: the scores are laid out as rows, the gradient comes back as planes."""
    g = torch.Generator().manual_seed(classes + k)
    index = torch.randint(-1, classes, (k, 5, 6), generator=g).to(DEV)
    check_distill(rand(classes, 5, 6) * 2, rand(k, 5, 6), index, 1.0, 0)
    leaf = rand(classes, 5, 6).requires_grad_(True)
    (d,) = torch.autograd.grad(losses.distill_loss(leaf, rand(k, 5, 6), index, class_dim=0), leaf)
    assert d.shape == leaf.shape


def test_captured_and_replayed_at_size():
    """As many positions as take the general sort, rows of an odd length, a mean that is counted in a launch of its own."""
    n, rows, dim = 20000, 900, 33

    def inputs(seed):
        t, ids = label(n, dim, 5, seed)
        return [tokens(n, rows, seed, 2.0, 0.05), rand(rows, dim, seed=seed), rand(dim, seed=seed), rand(dim, seed=seed + 1), t, ids]

    def step(index, table, w, b, t, ids):
        p = [x.detach().requires_grad_(True) for x in (table, w, b)]
        z = features.layer_norm(features.embedding(index, p[0], 2.0), p[1], p[2])
        value, d = losses.distill_loss_raw(z, t, ids, 2.0)
        return [value, *torch.autograd.grad(z, p, d)]

    sets = [inputs(k) for k in range(3)]
    want = [step(*v) for v in sets]
    held = [x.clone() for x in sets[0]]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(*held)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(*held)
    for k in (1, 2, 0, 2, 1):
        for a, b in zip(held, sets[k]):
            a.copy_(b)
        graph.replay()
        step(*sets[(k + 1) % 3])
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want[k])), k
