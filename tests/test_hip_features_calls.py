"""Calls of embedding, layer_norm and distill_loss beside the ordinary ones."""
import math

import pytest
import torch
import torch.autograd.forward_ad as fwd

from event_3dgs_amd import features, losses

pytestmark = pytest.mark.gpu
DEV = "cuda"


def rand(*shape, seed=0):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed + sum(shape))).to(DEV)


def test_forward_mode_is_refused():
    """A result without a tangent would be read as a derivative of zero."""
    x, w, d = rand(4, 6), rand(6), rand(4, 6, seed=1)
    t, ids = rand(4, 2), torch.zeros(4, 2, dtype=torch.int64, device=DEV)
    for grad in (False, True):
        with fwd.dual_level():
            dual = fwd.make_dual(x.clone().requires_grad_(grad), d)
            dual_w = fwd.make_dual(w.clone().requires_grad_(grad), d[0])
            dual_t = fwd.make_dual(t.clone(), d[:, :2])
            calls = [lambda: features.embedding(ids, dual), lambda: features.layer_norm(dual), lambda: features.layer_norm(x, dual_w),
                     lambda: features.layer_norm(x, None, dual_w), lambda: losses.distill_loss(dual, t, ids),
                     lambda: losses.distill_loss(x, dual_t, ids)]
            for k, call in enumerate(calls):
                for mode in (torch.enable_grad(), torch.no_grad()):
                    with mode, pytest.raises(RuntimeError, match="forward-mode"):
                        call()
                        pytest.fail("call %d was not refused" % k)
            # without autograd: value and gradient of the primal
            value, grad_x = losses.distill_loss_raw(dual, t, ids)
            assert fwd.unpack_dual(value).tangent is None and fwd.unpack_dual(grad_x).tangent is None
            features.layer_norm(x, w)                            # (no tangent among the inputs)
    leaf = x.clone().requires_grad_(True)
    for call in (lambda: features.embedding(ids, leaf), lambda: features.layer_norm(leaf), lambda: losses.distill_loss(leaf, t, ids)):
        with fwd.dual_level():                                   # ... or of the gradient that comes back
            y = call()
            with pytest.raises(RuntimeError, match="forward-mode"):
                torch.autograd.grad(y, leaf, fwd.make_dual(torch.ones_like(y), torch.ones_like(y)))


def peak_of(call):
    torch.cuda.synchronize()
    base = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    out = call()
    torch.cuda.synchronize()
    return out, torch.cuda.max_memory_allocated() - base


def test_layer_norm_forms_the_gradients_asked_for():
    x, w, b = (rand(*s).requires_grad_(True) for s in ((20000, 256), (256,), (256,)))
    d = rand(20000, 256, seed=1)
    # dx, and the partial sums of the parameters' gradients (at most 1024 pairs of rows).  The allocator keeps up to 1 MiB behind
    # an allocation with it (it cuts a block only where more is left): the 20480000 bytes of dx are 20971520 in its steps of 2 MiB.
    size, sums = 20000 * 256 * 4 + 2 ** 20, 1024 * 2 * 256 * 4 + 2 ** 20
    full = torch.autograd.grad(features.layer_norm(x, w, b), (x, w, b), d)
    y = features.layer_norm(x, w, b)
    for wanted in ((0,), (1,), (2,), (0, 2), (1, 2)):
        got, peak = peak_of(lambda: torch.autograd.grad(y, [(x, w, b)[k] for k in wanted], d, retain_graph=True))
        assert all(torch.equal(g, full[k]) for g, k in zip(got, wanted))
        assert peak <= (size if 0 in wanted else 0) + (sums if wanted != (0,) else 0) + 65536, wanted
    y = features.layer_norm(x, None, b)                          # (the bias in the weight's place among the gradients)
    (got,), peak = peak_of(lambda: torch.autograd.grad(y, b, d))
    assert torch.equal(got, full[2]) and peak <= sums + 65536


@pytest.mark.parametrize("dim", [66, 65])
def test_embedding_past_one_launch(dim):
    """More workgroups than one launch takes (2^32 threads): 2^36 values and some more, in packs of 4 bytes and one by one."""
    n = 2 ** 36 // dim + 1003
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < (2 * dim + 8) * n:
        pytest.skip("needs 146 GB of device memory")
    table = rand(7, dim).half()
    index = (torch.arange(n, dtype=torch.int32, device=DEV) * 5).remainder_(7)
    out = features.embedding(index, table)
    for first in (0, n // 2, 2 ** 35 // dim - 500, n - 1000):    # (the middle, where another launch may begin, the end)
        assert torch.equal(out[first:first + 1000], table[index[first:first + 1000]]), first
    del out, index
    torch.cuda.empty_cache()


# ------------------------------------------------------------------------------------------------ the largest counts
def test_embedding_of_the_most_positions():
    n = 2 ** 31 - 2
    index = torch.arange(n, dtype=torch.int32, device=DEV).remainder_(3)
    index[-1] = -1
    table = torch.tensor([[1.0], [2.0], [3.0], [4.0]], device=DEV).half().requires_grad_(True)
    out = features.embedding(index, table)
    assert out.shape == (n, 1) and out[-5:, 0].tolist() == [float((n - 5 + i) % 3 + 1) for i in range(4)] + [0.0]
    assert out[n // 2:n // 2 + 3, 0].tolist() == [float((n // 2 + i) % 3 + 1) for i in range(3)]
    del out
    table = table.detach().float().requires_grad_(True)
    out = features.embedding(index, table)
    (grad,) = torch.autograd.grad(out, table, torch.full((1, 1), 2.0 ** -10, device=DEV).expand(n, 1))
    counts = [(n - 1 - k + 2) // 3 for k in range(3)]
    # 128 equal terms are summed exactly, then up to 87382 partial sums in a row (below 2^24 * 2^-10: exactly too), then 64 of them
    for got, count in zip(grad[:, 0].tolist(), counts + [0]):
        assert abs(got - count * 2.0 ** -10) <= 70 * 2.0 ** -24 * count * 2.0 ** -10
    del out, index
    torch.cuda.empty_cache()


def test_layer_norm_of_more_rows_than_31_bits():
    n = 2 ** 31 + 5
    x = torch.zeros(n, 2, dtype=torch.float16, device=DEV)
    x[-9:] = ((rand(9, 2) * 4).round() / 4).half()               # (quarters: mean and variance are exact, in any order)
    x[n // 2] = torch.tensor([0.5, -2.0], device=DEV)
    out = features.layer_norm(x.requires_grad_(True))
    assert torch.equal(out[-9:], features.layer_norm(x.detach()[-9:])) and torch.equal(out[n // 2], features.layer_norm(x.detach()[n // 2]))
    d = torch.zeros_like(out)
    d[-2, 0], d[-1, 1] = 1.0, 2.0                                # (one term to each sum)
    (dx,) = torch.autograd.grad(out, x, d)
    last = x.detach()[-2:].requires_grad_(True)
    (want,) = torch.autograd.grad(features.layer_norm(last), last, d[-2:])
    assert torch.equal(dx[-2:], want) and want.count_nonzero() > 0 and dx[-1000:-2].count_nonzero() == 0
    del out, dx, d, x
    torch.cuda.empty_cache()


@pytest.mark.parametrize("planes", [False, True])
def test_distill_of_the_most_rows(planes):
    """Two equal scores, one of them listed: every row is log 2, its gradient -1/2 and 1/2."""
    n = 2 ** 31 - 4
    z = torch.zeros((2, n) if planes else (n, 2), dtype=torch.float16, device=DEV).requires_grad_(True)
    t = torch.zeros(1, 1, device=DEV).expand((1, n) if planes else (n, 1))
    ids = torch.zeros(1, 1, dtype=torch.int32, device=DEV).expand(t.shape)
    for how in ("mean", "sum"):
        value, d = losses.distill_loss_raw(z, t, ids, reduction=how, class_dim=0 if planes else 1)
        # a thread adds up n / (4096 * 256) rows one by one, a workgroup its threads in a tree; the rest is 64 bits
        want = math.log(2) * (1 if how == "mean" else n)
        assert abs(value.item() - want) <= (n / 2 ** 20 + 20) * 2.0 ** -24 * want
        if how == "sum":
            both = d if planes else d.t()
            for part in (both[:, :1000], both[:, n // 2:n // 2 + 1000], both[:, -1000:]):
                assert (part[0] == -0.5).all() and (part[1] == 0.5).all()
        del d
    loss = losses.distill_loss(z, t, ids, reduction="sum", class_dim=0 if planes else 1)
    (d,) = torch.autograd.grad(loss, z)
    both = d if planes else d.t()
    assert (both[0, -1000:] == -0.5).all() and (both[1, -1000:] == 0.5).all()
    del z, d, both, loss
    torch.cuda.empty_cache()


def test_first_call_captured():
    """Calls whose kernels nothing has launched before: one graph, replayed on other inputs."""
    shapes = [(1031, 1541), (1029, 12294), (67, 8194), (130, 40010)]         # (no other test takes these)

    def inputs(seed):
        v = []
        for k, s in enumerate(shapes):
            g = torch.Generator().manual_seed(seed + k)
            index = torch.randint(-1, 9, (s[0],), generator=g).to(DEV)
            v.append([index, rand(9, s[1], seed=seed).half(), rand(s[1], seed=seed).half(), rand(s[1], seed=seed + 1).half(),
                      rand(s[0], 3, seed=seed), torch.randint(0, s[1], (s[0], 3), generator=g).to(DEV)])
        return v

    def step(v):
        out = []
        for index, table, w, b, t, ids in v:
            p = [x.detach().requires_grad_(True) for x in (table, w, b)]
            z = features.layer_norm(features.embedding(index, p[0]), p[1], p[2])
            loss = losses.distill_loss(z, t, ids, 2.0, "sum")
            out += [loss.detach(), *torch.autograd.grad(loss, p)]
        return out

    held = inputs(0)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        out = step(held)
    for seed in (1, 2, 0, 3):
        new = inputs(seed)
        for a, b in zip(sum(held, []), sum(new, [])):
            a.copy_(b)
        graph.replay()
        want = step(new)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want)), seed
