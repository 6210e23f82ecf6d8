"""Block selection where the scores are hard to tell apart: below the normal range, neighbours,
of extreme spread.  A selection has one right value and is compared for equality."""
import pytest
import torch

from nntile_b200.sdpa import KVPages, paged_select
from test_gpu_paged import chosen, gen, ints

pytestmark = pytest.mark.gpu


def select_of(low, high, q, D, S, first=0, last=0, missing=()):
    """Selection among len(low) blocks whose bounds differ in their first element only."""
    count, P = len(low), 16
    pages = KVPages.empty(count, P, 1, D, bounds=True)
    pages.bounds[:, 0, 0, 0] = low.to(torch.bfloat16)
    pages.bounds[:, 0, 1, 0] = high.to(torch.bfloat16)
    table = torch.randperm(count, generator=gen(count), device="cuda", dtype=torch.int32).reshape(1, -1)
    for x in missing:
        table[0, x] = -1
    query = torch.zeros((1, 2, 1, 1, D), dtype=torch.bfloat16, device="cuda")
    query[0, :, 0, 0, 0] = q
    lens = ints(count*P)
    got = paged_select(query, pages, lens, table, S, first, last)
    if not missing:
        assert torch.equal(got, chosen(query, pages.bounds, lens, table, P, S, first, last))
    return got, table


@pytest.mark.parametrize("D", [64, 128, 256, 20])        # the tensor instruction, and without it
@pytest.mark.parametrize("S", [1, 100, 599])
def test_scores_below_the_normal_range(D, S):
    count = 600
    g = gen(D + S)
    tiny = 2.0**-74                                      # times 2^-75: the smallest float
    for top in (1, 2, 4, 5, 250):
        x = torch.randint(top - 1, top + 1, (count,), generator=g, device="cuda").float()*tiny
        select_of(x, x, 2.0**-75, D, S)
        select_of(-x, x, -2.0**-75, D, S)
    x = torch.randint(0, 256, (count,), generator=g, device="cuda").float()*tiny
    select_of(x, x, 2.0**-75, D, S, 1 if S > 1 else 0, 0)
    select_of(x, x, 2.0**-60, D, S)


@pytest.mark.parametrize("D", [64, 20])
@pytest.mark.parametrize("count", [700, 3000])
def test_scores_of_extreme_spread(D, count):
    g = gen(count)
    x = torch.randn(count, generator=g, device="cuda")
    wide = x*torch.exp2(torch.randint(-130, 120, (count,), generator=g, device="cuda").float())
    for S in (1, 300, 650):
        select_of(wide, wide, 1.0, D, S)
        select_of(x, x, 2.0**-100, D, S)                 # a range below 2^-96
        one = torch.full((count,), 1.0, device="cuda")
        one[count//2:] += 2.0**-7                        # two values, one step apart
        select_of(one, one, 1.0, D, S)
        select_of(one, one, 2.0**-110, D, S)
        one[7] = 2.0**100
        one[9] = -2.0**100
        select_of(one, one, 1.0, D, S)


def test_blocks_without_a_page_among_close_scores():
    count = 900
    x = torch.randint(0, 2, (count,), generator=gen(1), device="cuda").float()*2.0**-74
    for D in (64, 20):
        missing = [0, 5, 450, 899]
        got, _ = select_of(x, x, 2.0**-75, D, count - 4, missing=missing)
        assert sorted(set(range(count)) - set(got[0, 0].tolist())) == missing
