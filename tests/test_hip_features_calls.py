"""Calls of embedding, layer_norm and distill_loss beside the ordinary ones."""
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
