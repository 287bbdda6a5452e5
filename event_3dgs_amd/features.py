"""Rows of learned features: lookup in a shared table and layer norm, each with its gradient.

The pieces of a feature field on the Gaussians beside their own parameters: a table of rows that many Gaussians share
(compressed colour coefficients, identity or semantic codes), looked up by `embedding`, normalised by `layer_norm` in front
of a decoder, and trained through the rasteriser (renderer.render(override_color=...)) or against a teacher's class scores
(losses.distill_loss).  They take a batch of any size, a single row included.

float32, float16 and bfloat16; sums and statistics are fp32, every result is rounded once.  No CPU path.  The order of
every sum is fixed by sizes, strides and alignment: the same call gives the same bits.  Work is enqueued on the current stream
of the tensors' device (whichever device is current) and may be captured into a graph; the gradients are differentiable once
(a call under create_graph raises), and forward-mode derivatives are refused.
"""
from . import _lib

_EXT = None


def _ext():
    """The compiled torch extension that holds the autograd nodes.  Raises when it has not been built."""
    global _EXT
    if _EXT is None:
        _lib.lib()                                      # loud failure if the HIP library itself is missing
        try:
            from diff_gaussian_rasterization import _C_native
        except ImportError as e:
            raise _lib.HipLibraryError(
                "diff_gaussian_rasterization._C_native not found: build it with "
                "`python -c 'import __graft_entry__ as g; g.build()'`.  These operators have no CPU fallback.") from e
        if _C_native.abi_version() != _lib.ABI_VERSION or not hasattr(_C_native, "embedding"):
            raise _lib.HipLibraryError("diff_gaussian_rasterization._C_native does not match libe3dgs_hip.so; rebuild")
        _EXT = _C_native
    return _EXT


def embedding(index, table, scale=1.0):
    """scale * table[index]: rows of `table` (rows, dim) for an int32 / int64 `index` of any shape -> index.shape + (dim,).

    An index below 0 stands for "no row": zeros, no gradient.  One at or past the table's end gives a row of NaN (and no
    gradient): only the device sees it, and the call does not wait for the device.  The gradient of the table adds up the
    rows of each index in their order (positions sorted by index, no atomics)."""
    return _ext().embedding(index, table, float(scale))


def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """(x - mean) / sqrt(var + eps) * weight + bias over the last dimension of x; weight / bias: (dim,) of one type (x's own,
    or another of the three), or None."""
    return _ext().layer_norm(x, weight, bias, float(eps))
