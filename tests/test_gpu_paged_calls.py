"""Calls of the paged functions as the documentation allows them: empty ones, and by either of the
two ways from the tensors to the library."""
import pytest
import torch

from nntile_b200 import sdpa
from nntile_b200.sdpa import (KVPages, PagedKVCache, paged_append, paged_decode, paged_gather,
                              paged_select)
from test_gpu_paged import DT, gen, ints, make_table, randn

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


def all_calls(dtype, e4m3, float8=False):
    """Every paged function once, in each of its forms: what they answer and what they write."""
    g, dt = gen(7), DT[dtype]
    H, B, D, G, P = 2, 3, 64, 4, 16
    lens, new = [0, 17, 300], [40, 1, 5]
    ends = [a + b for a, b in zip(lens, new)]
    N = sum(-(-x//P) for x in ends) + 1
    pages = KVPages.empty(N, P, H, D, dt, e4m3, bounds=True)
    table = make_table(g, ends, P, N)
    status = ints(0)
    rows = [randn(g, H, B, 300, D).to(dt) for _ in range(2)]
    paged_append(pages, ints(0, 0, 0), table, *rows, ints(*lens), status)
    rows = [randn(g, H, B, 40, D).to(dt) for _ in range(2)]
    if float8:
        pages = KVPages(pages.k.view(torch.float8_e4m3fn), pages.v.view(torch.float8_e4m3fn),
                        pages.k_scales, pages.v_scales, pages.bounds)
    paged_append(pages, ints(*lens), table, *rows, ints(*new))
    at = ints(*ends)
    ko, vo = (torch.full((H, B, 310, D), 3.0, dtype=dt, device="cuda") for _ in range(2))
    paged_gather(pages, at, table, ko, vo, status)
    q = randn(g, H, G, B, 1, D).to(dt)
    ws = torch.empty(1 << 22, dtype=torch.uint8, device="cuda")
    sel = paged_select(q, pages, at, table, 6)
    sel2 = torch.zeros((H, B, 4), dtype=torch.int32, device="cuda")
    assert paged_select(q, pages, at, table, 4, 0, 2, sel2, ws, status) is sel2
    lse = torch.zeros((H, G, B), device="cuda")
    dense = paged_decode(q, pages, at, table)
    out = torch.zeros_like(q)
    assert paged_decode(q, pages, at, table, sel, out, lse, ws, status) is out
    wrong = ints(5000, 5000, 5000)
    paged_decode(q, pages, wrong, table, status=status)
    state = [pages.k, pages.v, pages.bounds] + ([pages.k_scales, pages.v_scales] if e4m3 else [])
    return [t.contiguous().view(torch.uint8) for t in state + [ko, vo, sel, sel2, dense, out, lse, status]]


@pytest.mark.parametrize("dtype,e4m3,float8", [("bf16", False, False), ("fp16", False, False),
                                               ("bf16", True, False), ("fp16", True, True)])
def test_both_ways_to_the_library_give_the_same(monkeypatch, dtype, e4m3, float8):
    """With the extension module and without it, bit for bit."""
    assert sdpa._paged_torch is not None
    with_module = all_calls(dtype, e4m3, float8)
    monkeypatch.setattr(sdpa, "_paged_torch", None)
    for a, b in zip(with_module, all_calls(dtype, e4m3, float8)):
        assert torch.equal(a, b)


def test_the_cache_object_without_the_module(monkeypatch):
    monkeypatch.setattr(sdpa, "_paged_torch", None)
    g = gen(8)
    cache = PagedKVCache(30, 16, 2, 2, 64, e4m3=True, bounds=True)
    for n in (50, 1, 20):
        cache.append(randn(g, 2, 2, n, 64).bfloat16(), randn(g, 2, 2, n, 64).bfloat16(), [n, n//2])
    q = randn(g, 2, 4, 2, 1, 64).bfloat16()
    bare = [cache.read()[0], cache.decode(q), cache.decode(q, num_selected=3)]
    monkeypatch.undo()
    for a, b in zip(bare, [cache.read()[0], cache.decode(q), cache.decode(q, num_selected=3)]):
        assert torch.equal(a, b)


def test_tensors_of_another_layout_are_refused_by_both(monkeypatch):
    pages = KVPages.empty(8, 16, 2, 64, bounds=True)
    table = torch.arange(8, dtype=torch.int32, device="cuda").reshape(1, 8)
    q = torch.zeros((2, 4, 1, 1, 64), dtype=torch.bfloat16, device="cuda")
    spread = torch.zeros((2, 4, 1, 1, 128), dtype=torch.bfloat16, device="cuda")[..., ::2]
    wide = torch.zeros((1, 16), dtype=torch.int32, device="cuda")[:, ::2]
    for module in (sdpa._paged_torch, None):
        monkeypatch.setattr(sdpa, "_paged_torch", module)
        for call in (lambda: paged_decode(spread, pages, ints(9), table),
                     lambda: paged_decode(q, pages, ints(9), wide),
                     lambda: paged_decode(q, pages, ints(9), table, out=spread),
                     lambda: paged_select(spread, pages, ints(9), table, 2),
                     lambda: paged_append(pages, ints(9), table, spread[:, :1, 0], spread[:, :1, 0]),
                     lambda: paged_decode(q, pages, ints(9).cpu(), table),
                     lambda: paged_decode(q, pages, ints(9), table, lse_out=torch.zeros(8)),
                     lambda: paged_gather(pages, ints(9), table, spread[:, :1, 0], spread[:, :1, 0])):
            with pytest.raises(ValueError):
                call()
