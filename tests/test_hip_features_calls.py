"""Calls of embedding, layer_norm and distill_loss beside the ordinary ones."""
import pytest
import torch

from event_3dgs_amd import features

pytestmark = pytest.mark.gpu
DEV = "cuda"


def rand(*shape, seed=0):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed + sum(shape))).to(DEV)


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
