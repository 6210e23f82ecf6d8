"""Calls of the paged functions as the documentation allows them: empty ones, and by either of the
two ways from the tensors to the library."""
import pytest
import torch

from nntile_b200.sdpa import KVPages, paged_decode, paged_select
from test_gpu_paged import ints

pytestmark = pytest.mark.gpu


def test_no_query_heads_select_nothing():
    pages = KVPages.empty(8, 16, 2, 64, bounds=True)
    q = torch.zeros((2, 0, 1, 1, 64), dtype=torch.bfloat16, device="cuda")
    table = torch.arange(8, dtype=torch.int32, device="cuda").reshape(1, 8)
    stale = torch.full((2, 1, 4), 12345, dtype=torch.int32, device="cuda")
    del stale                                  # the allocator hands this memory out again
    got = paged_select(q, pages, ints(100), table, 4)
    assert bool((got == -1).all())
    given = torch.full((2, 1, 4), 7, dtype=torch.int32, device="cuda")
    assert paged_select(q, pages, ints(100), table, 4, out=given) is given and bool((given == 7).all())
    assert paged_decode(q, pages, ints(100), table, got).shape == q.shape
