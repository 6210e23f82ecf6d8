"""Paged key/value cache on the GPU, through the public functions, against plain
implementations in 64 bits.

What is stored (rows, codes, exponent bytes, bounds, selections) has one right value and is
compared for equality.  For attention, with u the half step of the output's type
(bf16 2^-8, fp16 2^-11 relative):

  a score is a sum of `head` exact products in 32 bits and two scalings: off by at most
    ds = (head + 16) * 2^-23 * sum_d |q_d||k_d| / sqrt(head)   (a product of 16- or 22-bit
    factors rounds once at most; a truncating accumulator loses 2^-23 of the running sum a
    step, hence 2^-23 and not 2^-24; a query brought to another 16-bit format loses at most
    2^-24 of its largest element, less than one of the 16 spare steps);
  weights are off by the factor exp(2 ds) (score and maximum), by 2^-16 (two 16-bit parts, an
    exponential of 2^-22) and sums of N terms by N * 2^-24, numerator and denominator each,
so |out - exact| <= u*|exact| + max|v| * (4 ds + 2^-15 + N * 2^-23), and the logarithm of the
sum is off by at most 2 ds + 2^-21 * (1 + |lse|) + N * 2^-23."""
import math

import pytest
import torch

from nntile_b200 import _lib, ops, sdpa
from nntile_b200.sdpa import (KVPages, PagedKVCache, paged_append, paged_decode, paged_gather,
                              paged_select)

pytestmark = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "fp16": torch.float16}
BAD_PAGE, BAD_LENGTH, BAD_BLOCK = 1, 2, 4


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(g, *shape):
    return torch.randn(shape, generator=g, device="cuda")


def ints(*values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def two_to(e):
    """2^e in 64 bits, by its bits."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def decoded(codes, scales):
    """Values of 8-bit pages in 64 bits, from the format."""
    c = codes.view(torch.uint8).long()
    e, m = (c >> 3) & 15, (c & 7).double()
    v = torch.where(e == 0, m*2.0**-9, (8 + m)*two_to(e - 10))
    v = torch.where((c & 127) == 127, math.nan, v)
    v = torch.where(c >= 128, -v, v)
    return v*two_to(scales.long() - 127)[..., None]


def quantised(x):
    """Row-wise e4m3 of 64-bit rows: (values it stands for, exponent byte)."""
    fin = torch.where(x.isfinite(), x, 0.0)
    amax = fin.abs().amax(-1)
    e = torch.zeros_like(amax, dtype=torch.long) - 126
    for _ in range(260):                      # the smallest e >= -126 with amax <= 448 * 2^e
        too_big = amax > 448*two_to(e)
        if not bool(too_big.any()):
            break
        e = e + too_big.long()
    e = torch.where(amax == 0, 0, e)
    y = fin*two_to(-e)[..., None]
    grain = two_to(torch.frexp(y.abs().clamp(min=2.0**-6)).exponent - 1 - 3)
    v = torch.round(y/grain)*grain*two_to(e)[..., None]
    return torch.where(x.isfinite(), v, math.nan), e + 127


def stored(pages, which):
    """(k or v, 64 bits) of the whole pool."""
    t = pages.k if which == "k" else pages.v
    if not pages.e4m3:
        return t.double()
    return decoded(t, pages.k_scales if which == "k" else pages.v_scales)


def make_pool(g, N, P, H, D, dtype, e4m3, bounds=False):
    """A pool full of old values."""
    pages = KVPages.empty(N, P, H, D, dtype, e4m3, bounds)
    for t in (pages.k, pages.v):
        x = randn(g, N, H, P, D)
        t.copy_((x*100).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8) if e4m3
                else x.to(dtype))
    if e4m3:
        for s in (pages.k_scales, pages.v_scales):
            s.copy_(torch.randint(117, 122, s.shape, generator=g, device="cuda"))
    if bounds:
        k = stored(pages, "k")
        pages.bounds.copy_(torch.stack([k.amin(2), k.amax(2)], 2).to(dtype))
    return pages


def make_table(g, lengths, P, N, spare=1):
    """Random distinct pages for every sequence, -1 behind them."""
    need = [-(-n//P) for n in lengths]
    wide = max(need) + spare
    order = torch.randperm(N, generator=g, device="cuda").tolist()
    rows = []
    for n in need:
        rows.append([order.pop() for _ in range(n)] + [-1]*(wide - n))
    return torch.tensor(rows, dtype=torch.int32, device="cuda")


def same(a, b):
    """Equal values; NaN equals NaN."""
    return bool(((a == b) | (a.isnan() & b.isnan())).all())


# ---------------------------------------------------------------------------- append, gather

@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("D,P,H,starts,news", [
    (128, 16, 2, [0, 5, 16, 31], [16, 1, 17, 0]),
    (64, 64, 3, [63, 64], [130, 1]),
    (256, 16, 1, [7], [1]),
    (80, 32, 2, [0, 40], [33, 64]),
    (24, 5, 2, [4, 9, 10], [11, 1, 3]),
    (20, 16, 1, [3, 0], [20, 7]),            # rows that are not a multiple of 16 bytes
    (1, 1, 2, [2, 0], [3, 1]),
])
def test_append_and_gather(D, P, H, starts, news, e4m3, dtype):
    dt, g = DT[dtype], gen(D + P)
    B, n = len(starts), max(news)
    ends = [a + b for a, b in zip(starts, news)]
    N = sum(-(-e//P) for e in ends) + 2
    pages = make_pool(g, N, P, H, D, dt, e4m3, bounds=True)
    table = make_table(g, ends, P, N)
    k, v = randn(g, H, B, n, D).to(dt), (3*randn(g, H, B, n, D)).to(dt)
    want = {w: stored(pages, w) for w in "kv"}
    scales = {"k": pages.k_scales, "v": pages.v_scales}
    want_scales = {w: None if s is None else s.clone() for w, s in scales.items()}
    want_bounds = pages.bounds.double()
    for b in range(B):
        for i in range(news[b]):
            at = starts[b] + i
            page, off = int(table[b, at//P]), at % P
            for w, src in (("k", k), ("v", v)):
                row = src[:, b, i].double()
                if e4m3:
                    row, byte = quantised(row)
                    want_scales[w][page, :, off] = byte.to(torch.uint8)
                want[w][page, :, off] = row
            row = want["k"][page, :, off].to(dt).double()
            if off == 0:
                want_bounds[page] = torch.stack([row, row], 1)
            else:
                want_bounds[page, :, 0] = torch.minimum(want_bounds[page, :, 0], row)
                want_bounds[page, :, 1] = torch.maximum(want_bounds[page, :, 1], row)
    status = ints(0)
    paged_append(pages, ints(*starts), table, k, v, ints(*news), status)
    for w in "kv":
        assert same(stored(pages, w), want[w])
        if e4m3:
            assert torch.equal(scales[w], want_scales[w])
    assert same(pages.bounds.double(), want_bounds)
    # and back, into buffers that are longer than any sequence
    ko = torch.full((H, B, max(ends) + 3, D), 7.0, dtype=dt, device="cuda")
    vo = ko.clone()
    paged_gather(pages, ints(*ends), table, ko, vo, status)
    for w, got in (("k", ko), ("v", vo)):
        for b in range(B):
            rows = want[w][table[b, :-(-ends[b]//P)].long()].transpose(0, 1).reshape(H, -1, D)
            assert same(got[:, b, :ends[b]].double(), rows[:, :ends[b]].to(dt).double())
            assert bool((got[:, b, ends[b]:] == 7.0).all())
    assert int(status) == 0


def test_append_of_equal_rows_without_new_lens_leaves_the_rest():
    g = gen(1)
    pages = make_pool(g, 6, 16, 2, 64, torch.bfloat16, False)
    before = pages.k.clone()
    table = ints(3, 1, 0, 5).reshape(2, 2)
    k = randn(g, 2, 2, 4, 64).bfloat16()
    paged_append(pages, ints(14, 2), table, k, k)
    want = before.clone()
    want[3, :, 14:16], want[1, :, :2] = k[:, 0, :2], k[:, 0, 2:]
    want[0, :, 2:6] = k[:, 1]
    assert torch.equal(pages.k, want)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("D", [128, 20])
def test_quantiser_at_its_edges(dtype, D):
    """Rows of zeros, of the type's largest and smallest values, a largest magnitude just at
    and just above what a scale holds, infinities and NaN."""
    dt = DT[dtype]
    fi = torch.finfo(dt)
    g = gen(3)
    x = randn(g, 12, D)
    x[0] = 0.0
    x[1] = fi.max*torch.sign(x[1])
    x[2] = fi.smallest_normal*fi.eps*torch.randint(-3, 4, (D,), generator=g, device="cuda")
    x[3] *= fi.smallest_normal
    x[4, 0] = 448.0
    x[4, 1:] = torch.linspace(-448, 448, D - 1)
    x[5, 0] = 450.0 if dtype == "bf16" else 448.25
    x[5, 1:] = torch.linspace(-448, 448, D - 1)
    x[6, 3] = math.inf
    x[7, 3], x[7, 4] = -math.inf, math.nan
    x[8] = math.nan
    x[9] = -0.0
    x[10] = torch.arange(D)*2.0**-9 + 2.0**-10              # ties below the normal range
    x[10, 0] = 448.0
    x[11] = 1e-3*x[11]
    rows = x.to(dt)
    pages = KVPages.empty(1, 12, 1, D, dt, e4m3=True)
    paged_append(pages, ints(0), ints(0).reshape(1, 1), rows.reshape(1, 1, 12, D),
                 rows.flip(0).reshape(1, 1, 12, D).contiguous())
    want, byte = quantised(rows.double())
    assert torch.equal(pages.k_scales[0, 0], byte.to(torch.uint8))
    assert same(stored(pages, "k")[0, 0], want)
    assert same(stored(pages, "v")[0, 0], want.flip(0))


def test_what_does_not_fit_is_dropped_and_reported():
    g = gen(4)
    for e4m3 in (False, True):
        pages = make_pool(g, 4, 16, 2, 64, torch.bfloat16, e4m3)
        before = stored(pages, "k")
        k = randn(g, 2, 3, 5, 64).bfloat16()
        table = ints(0, 1, 2, 9, -7, 3).reshape(3, 2)       # two entries outside the pool
        status = ints(0)
        paged_append(pages, ints(30, 14, 2), table, k, k, None, status)
        got = stored(pages, "k")
        want = before.clone()
        new = k.double() if not e4m3 else quantised(k.double())[0]
        want[1, :, 14:16] = new[:, 0, :2]                   # three rows past the table
        want[2, :, 14:16] = new[:, 1, :2]                   # three on page 9
        assert same(got, want)
        assert int(status) == BAD_PAGE | BAD_LENGTH
        status.zero_()
        paged_append(pages, ints(-3, 200, 0), ints(0, 1, 2, 3, 3, 3).reshape(3, 2), k, k,
                     ints(0, 1, 0), status)
        assert same(stored(pages, "k"), want) and int(status) == BAD_LENGTH
        status.zero_()
        out = torch.zeros((2, 3, 20, 64), dtype=torch.bfloat16, device="cuda")
        paged_gather(pages, ints(32, 17, 3), table, out, out.clone(), status)
        assert int(status) == BAD_PAGE | BAD_LENGTH
        assert same(out[:, 1, :16].double(), stored(pages, "k")[2].bfloat16().double())
        assert bool((out[:, 1, 16:] == 0).all()) and bool((out[:, 2] == 0).all())


# ---------------------------------------------------------------------------------- decode

def attention(q, pages, lengths, table, selected=None):
    """(out, lse, largest ds, most terms, largest |v|), 64 bits, position by position lists."""
    H, G, B, _, D = q.shape
    P = pages.k.shape[2]
    K, V = stored(pages, "k"), stored(pages, "v")
    out = torch.zeros((H, G, B, 1, D), dtype=torch.float64, device="cuda")
    lse = torch.full((H, G, B), -math.inf, dtype=torch.float64, device="cuda")
    ds, terms, vmax = 0.0, 1, 0.0
    for b, n in enumerate(lengths.tolist()):
        for h in range(H):
            blocks = list(range(-(-n//P))) if selected is None else \
                [x for x in selected[h, b].tolist() if 0 <= x < -(-n//P)]
            k = [K[int(table[b, x]), h, :min(P, n - x*P)] for x in blocks]
            v = [V[int(table[b, x]), h, :min(P, n - x*P)] for x in blocks]
            if not k:
                continue
            k, v, qq = torch.cat(k), torch.cat(v), q[h, :, b, 0].double()
            s = qq @ k.T/math.sqrt(D)
            lse[h, :, b] = torch.logsumexp(s, -1)
            out[h, :, b, 0] = torch.softmax(s, -1) @ v
            ds = max(ds, (D + 16)*2.0**-23/math.sqrt(D)*float((qq.abs() @ k.abs().T).max()))
            terms, vmax = max(terms, len(k)), max(vmax, float(v.abs().max()))
    return out, lse, ds, terms, vmax


def check_attention(q, pages, lengths, table, selected=None):
    H, G, B, _, D = q.shape
    want, want_lse, ds, terms, vmax = attention(q, pages, lengths, table, selected)
    lse = torch.full((H, G, B), math.nan, dtype=torch.float32, device="cuda")
    status = ints(0)
    out = paged_decode(q, pages, lengths, table, selected, lse_out=lse, status=status)
    torch.cuda.synchronize()
    assert int(status) == 0
    half = torch.finfo(q.dtype).eps/2
    tol = half*want.abs() + vmax*(4*ds + 2.0**-15 + terms*2.0**-23) \
        + torch.finfo(q.dtype).smallest_normal*torch.finfo(q.dtype).eps
    assert bool(((out.double() - want).abs() <= tol).all()), \
        float(((out.double() - want).abs()/tol).max())
    empty = want_lse == -math.inf
    assert bool((lse[empty] == -math.inf).all())
    tol = 2*ds + 2.0**-21*(1 + want_lse[~empty].abs()) + terms*2.0**-23
    assert bool(((lse.double()[~empty] - want_lse[~empty]).abs() <= tol).all())
    return out, lse


def poison_tails(pages, lengths, table):
    """NaN in every position that no sequence has filled."""
    N, H, P, D = pages.k.shape
    live = torch.zeros((N, P), dtype=torch.bool, device="cuda")
    for b, n in enumerate(lengths.tolist()):
        for x in range(-(-n//P)):
            live[int(table[b, x]), :min(P, n - x*P)] = True
    dead = (~live)[:, None, :, None].expand(N, H, P, D)
    for t in (pages.k, pages.v):
        if pages.e4m3:
            t.masked_fill_(dead, 0x7F)
        else:
            t.masked_fill_(dead, math.nan)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("D,P,H,G,lengths", [
    (128, 16, 2, 4, [1, 15, 16, 17, 0, 333]),
    (128, 64, 1, 8, [64, 65, 63, 1000]),
    (64, 16, 3, 1, [129]),
    (64, 32, 2, 5, [0, 0]),
    (128, 16, 1, 9, [500, 3]),
    (128, 48, 2, 17, [97, 200]),             # more query heads than two tiles of eight
    (256, 16, 1, 2, [40, 700]),
    (80, 32, 2, 3, [31, 32, 33]),
    (96, 16, 2, 12, [250]),
    (16, 16, 2, 4, [77, 5]),
    (40, 16, 1, 4, [100]),                   # 16-bit rows of 80 bytes, 8-bit rows of 40
    (128, 5, 2, 4, [1, 4, 5, 6, 143]),       # pages that are no multiple of 16
    (100, 16, 1, 3, [50]),
    (7, 3, 1, 2, [10, 2]),
    (1, 1, 1, 1, [4]),
    (128, 16, 8, 4, [2048]),
    (128, 128, 1, 1, [5000, 2, 1200]),
    (256, 16, 2, 9, [300, 50]),              # two tiles of heads, each with a pass of its own
    (64, 16, 1, 1, [60001]),                 # one unit over every SM
    (64, 32, 8, 2, [(37*i) % 401 for i in range(40)]),       # many units, a warp takes several
    (64, 16, 8, 3, [(29*i) % 251 for i in range(40)]),       # and none is long enough to split
    (128, 32, 4, 3, [(211*i) % 977 for i in range(20)]),
    (128, 16, 4, 1, [1]*19 + [9000]),        # one long among short ones
])
def test_decode_against_64_bits(D, P, H, G, lengths, e4m3, dtype):
    dt, g = DT[dtype], gen(D*P + G)
    N = sum(-(-n//P) for n in lengths) + 2
    pages = make_pool(g, N, P, H, D, dt, e4m3)
    table = make_table(g, lengths, P, N)
    lens = ints(*lengths)
    poison_tails(pages, lens, table)
    q = (2*randn(g, H, G, len(lengths), 1, D)).to(dt)
    check_attention(q, pages, lens, table)


@pytest.mark.parametrize("B,H,G,D", [(2, 3, 2, 128), (8, 4, 2, 256), (31, 1, 3, 64), (33, 2, 2, 128),
                                     (64, 2, 1, 64), (65, 2, 1, 64)])
@pytest.mark.parametrize("lengths", ["even", "ragged", "one"])
def test_decode_cuts_units_into_pieces(B, H, G, D, lengths):
    """Few units of several lengths: shares that end with the units and shares that do not."""
    g = gen(100*B + D)
    P, n = 16, 700
    lens = [n]*B if lengths == "even" else [0]*(B - 1) + [5*n] if lengths == "one" else \
        [int(x) for x in torch.randint(0, 2*n, (B,), generator=torch.Generator().manual_seed(B))]
    num_pages = sum(-(-x//P) for x in lens) + 1
    pages = make_pool(g, num_pages, P, H, D, torch.bfloat16, False)
    table = make_table(g, lens, P, num_pages)
    q = randn(g, H, G, B, 1, D).bfloat16()
    check_attention(q, pages, ints(*lens), table)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("e4m3", [False, True])
def test_decode_with_far_apart_values(e4m3, dtype):
    """Rows of very different size: scores that dwarf the others early, late and in the
    middle, values over many binades, queries with tiny elements."""
    dt, g = DT[dtype], gen(9)
    D, P, H, G, lengths = 64, 16, 2, 4, [700, 333]
    N = sum(-(-n//P) for n in lengths)
    pages = KVPages.empty(N, P, H, D, dt, e4m3)
    table = make_table(g, lengths, P, N)
    n = max(lengths)
    size = torch.exp2(torch.randint(-9, 4, (H, 2, n, 1), generator=g, device="cuda").float())
    k = randn(g, H, 2, n, D)*size.clamp(max=1.0)
    k[:, :, 5] *= 4
    k[:, 0, 650] *= 4
    v = randn(g, H, 2, n, D)*size
    paged_append(pages, ints(0, 0), table, k.to(dt), v.to(dt), ints(*lengths))
    q = randn(g, H, G, 2, 1, D)
    q[..., ::3] *= 2.0**-14
    check_attention(q.to(dt), pages, ints(*lengths), table)


def test_decode_whose_scores_are_minus_infinity():
    """Keys of -inf against positive queries: no weight at all, and no NaN; one finite key
    among them takes everything."""
    D, P = 64, 16
    pages = KVPages.empty(2, P, 1, D)
    pages.k.fill_(-math.inf)
    pages.v.fill_(3.0)
    q = torch.ones((1, 2, 1, 1, D), dtype=torch.bfloat16, device="cuda")
    lse = torch.empty((1, 2, 1), device="cuda")
    table = ints(1, 0).reshape(1, 2)
    out = paged_decode(q, pages, ints(20), table, lse_out=lse)
    assert bool((out == 0).all()) and bool((lse == -math.inf).all())
    pages.k[0, 0, 2] = 0.5                                   # position 18
    pages.v[0, 0, 2] = -2.0
    out = paged_decode(q, pages, ints(20), table, lse_out=lse)
    assert bool((out == -2.0).all())
    assert bool(((lse - 0.5*D/8).abs() <= 2.0**-21*(1 + 0.5*D/8)).all())
    # a key of NaN reaches the output of its own sequence
    pages.k[0, 0, 2, 7] = math.nan
    assert bool(paged_decode(q, pages, ints(20), table).isnan().all())


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("D,P,G", [(128, 16, 4), (64, 32, 9), (72, 5, 3)])
def test_decode_of_selected_blocks(D, P, G, e4m3):
    g = gen(D + G)
    H, lengths = 2, [200, 3, 0, 77]
    N = sum(-(-n//P) for n in lengths) + 1
    pages = make_pool(g, N, P, H, D, torch.bfloat16, e4m3)
    table = make_table(g, lengths, P, N, spare=3)
    lens = ints(*lengths)
    poison_tails(pages, lens, table)
    q = randn(g, H, G, 4, 1, D).bfloat16()
    last = (lengths[0] - 1)//P
    sel = torch.full((H, 4, 6), -1, dtype=torch.int32, device="cuda")
    sel[0, 0] = ints(last, 0, -1, 3, -5, 1)                  # any order, holes, the ragged block
    sel[1, 0] = ints(2, 2, last, last, 2, -1)                # blocks listed more than once
    sel[0, 1] = ints(0, 1, -1, -1, -1, -1)                   # block 1 is behind the length
    sel[1, 2] = ints(0, 1, 2, 3, 4, 5)                       # nothing is filled
    sel[0, 3] = ints(-1, -1, -1, -1, -1, 0)
    check_attention(q, pages, lens, table, sel)              # sel[1, 1], sel[1, 3] select nothing


def test_decode_reports_what_it_leaves_out():
    g = gen(5)
    for D, P in ((64, 16), (20, 3)):
        pages = make_pool(g, 8, P, 1, D, torch.float16, False)
        q = randn(g, 1, 2, 3, 1, D).half()
        good = torch.tensor([[0, 1, -1], [2, 3, -1], [4, 5, 6]], dtype=torch.int32, device="cuda")
        want, want_lse, *_ = attention(q, pages, ints(2*P, P, 3*P), good)
        bad = torch.tensor([[0, 1, 77], [2, -4, 8], [4, 5, 6]], dtype=torch.int32, device="cuda")
        status = ints(0)
        out = paged_decode(q, pages, ints(3*P, 2*P, 2000), bad, status=status)
        assert int(status) == BAD_PAGE | BAD_LENGTH
        assert float((out.double() - want).abs().max()) < 0.02
        status.zero_()
        sel = ints(0, 1, 2, 0, 3, -1, 0, 1, 2147483647).reshape(1, 3, 3)
        out = paged_decode(q, pages, ints(2*P, P, -5), good, sel, status=status)
        assert int(status) == BAD_BLOCK | BAD_LENGTH
        assert float((out.double() - want)[:, :, :2].abs().max()) < 0.02
        assert bool((out[:, :, 2] == 0).all())


def test_decode_equals_the_contiguous_cache():
    """The same cache in pages and in one piece, by the framework's two decode paths."""
    g = gen(6)
    H, B, L, D, G = 2, 3, 777, 128, 4
    cache = sdpa.KVCache(L, H, B, D)
    paged = PagedKVCache(3*50, 16, H, B, D)
    for n in (700, 76, 1):
        k, v = randn(g, H, B, n, D).bfloat16(), randn(g, H, B, n, D).bfloat16()
        cache.append(k, v)
        paged.append(k, v)
    q = randn(g, H, G, B, 1, D).bfloat16()
    k, v = paged.read()
    assert torch.equal(k, cache.k) and torch.equal(v, cache.v)
    layer = sdpa.Sdpa(q, cache.k[:, None], cache.v[:, None])
    a = layer.forward_dynamic(q, None, None, kv_cache=cache)
    b = layer.forward_dynamic(q, None, None, kv_cache=paged)
    # the contiguous kernel keeps its weights in bf16: half a step each, and one of the output
    assert float((a.double() - b.double()).abs().max()) <= 2.0**-8*float(cache.v.abs().max())


# ---------------------------------------------------------------------------------- select

def chosen(q, bounds, lengths, table, P, S, first, last):
    H, G, B, _, D = q.shape
    out = torch.full((H, B, S), -1, dtype=torch.int32)
    for b, n in enumerate(lengths.tolist()):
        count = -(-n//P)
        if count == 0:
            continue
        bd = bounds[table[b, :count].long()].double()
        for h in range(H):
            s = torch.full((count,), -math.inf, dtype=torch.float64, device="cuda")
            for x in q[h, :, b, 0].double():
                s = torch.maximum(s, (x.clamp(min=0)*bd[:, h, 1] + x.clamp(max=0)*bd[:, h, 0])
                                  .sum(-1))
            s = torch.where(s.isnan(), math.inf, s).tolist()
            always = [i for i in range(count) if i < first or i >= count - last][:S]
            rest = sorted((i for i in range(count) if i not in always), key=lambda i: -s[i])
            pick = sorted(always + rest[:S - len(always)])
            out[h, b, :len(pick)] = torch.tensor(pick, dtype=torch.int32)
    return out.cuda()


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("D,P,H,G,lengths,S,first,last", [
    (128, 16, 2, 4, [1000, 17, 0, 333], 8, 1, 1),
    (64, 16, 3, 1, [5000], 33, 0, 0),
    (128, 32, 1, 8, [3000, 96, 97], 3, 1, 2),
    (128, 16, 2, 9, [700], 20, 0, 3),
    (80, 5, 2, 3, [444, 5], 6, 2, 0),
    (20, 16, 1, 17, [300], 5, 0, 1),
    (256, 16, 1, 2, [400], 1, 0, 0),
    (128, 16, 1, 4, [9000], 500, 1, 1),
    (64, 1, 1, 2, [3], 2, 0, 0),
    (128, 16, 1, 2, [64], 4, 2, 2),          # everything is taken
])
def test_select_against_64_bits(D, P, H, G, lengths, S, first, last, dtype):
    dt, g = DT[dtype], gen(D + S)
    N = sum(-(-n//P) for n in lengths) + 1
    pages = make_pool(g, N, P, H, D, dt, False, bounds=True)
    table = make_table(g, lengths, P, N)
    q = randn(g, H, G, len(lengths), 1, D).to(dt)
    lens, status = ints(*lengths), ints(0)
    got = paged_select(q, pages, lens, table, S, first, last, status=status)
    assert int(status) == 0
    assert torch.equal(got, chosen(q, pages.bounds, lens, table, P, S, first, last))


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_select_ties_and_near_ties(dtype):
    """Blocks that are the same, or whose scores differ by one part in 2^23 only: the sums
    decide exactly, equal ones go to the lowest block."""
    dt, g = DT[dtype], gen(12)
    D, P, H, G, S = 128, 16, 2, 4, 40
    count = 600
    pages = make_pool(g, count, P, H, D, dt, False, bounds=True)
    table = torch.randperm(count, generator=g, device="cuda", dtype=torch.int32).reshape(1, count)
    q = randn(g, H, G, 1, 1, D).to(dt)
    lens = ints(count*P)
    pages.bounds.copy_(pages.bounds[:1].expand_as(pages.bounds).clone())
    got = paged_select(q, pages, lens, table, S, 0, 0)
    assert torch.equal(got[0, 0], torch.arange(S, dtype=torch.int32, device="cuda"))
    # sizes far apart: a tiny element decides beneath terms that cancel in 32 bits
    q[..., :] = 1.0
    base = torch.zeros((D,), device="cuda")
    base[0], base[1] = 4096.0, -4096.0
    tiny = (torch.randint(0, 50, (count,), generator=g, device="cuda").float())*2.0**-14
    b = base.expand(count, D).clone()
    b[:, 2] = tiny
    pages.bounds.copy_(b[:, None, None].expand(count, H, 2, D).to(dt))
    assert torch.equal(paged_select(q, pages, lens, table, S, 0, 0),
                       chosen(q, pages.bounds, lens, table, P, S, 0, 0))
    assert torch.equal(paged_select(q, pages, lens, table, S, 3, 2),
                       chosen(q, pages.bounds, lens, table, P, S, 3, 2))


def test_select_with_nan_infinite_and_missing_pages():
    g = gen(13)
    D, P, H, G, count, S = 64, 16, 1, 2, 100, 6
    pages = make_pool(g, count, P, H, D, torch.bfloat16, False, bounds=True)
    pages.bounds[40, 0, :, 5] = math.nan
    pages.bounds[41, 0, 0, 5], pages.bounds[41, 0, 1, 5] = -math.inf, math.inf
    pages.bounds[42, 0] = -math.inf                          # 0 * inf: NaN as well
    table = torch.arange(count, dtype=torch.int32, device="cuda").reshape(1, count).clone()
    q = (randn(g, H, G, 1, 1, D).abs() + 0.1).bfloat16()
    lens, status = ints(count*P), ints(0)
    got = paged_select(q, pages, lens, table, S, 0, 0, status=status)
    assert int(status) == 0 and {40, 41, 42} <= set(got[0, 0].tolist())
    assert torch.equal(got, chosen(q, pages.bounds, lens, table, P, S, 0, 0))
    table[0, 3] = 5000
    got = paged_select(q, pages, lens, table, count - 1, 0, 0, status=status)
    assert int(status) == BAD_PAGE
    # behind every block that has a page
    assert sorted(set(range(count)) - set(got[0, 0].tolist())) == [3]


def test_select_without_a_pool():
    """Every page is missing: the lowest blocks, reported, nothing read."""
    for D in (64, 20):
        pages = KVPages.empty(0, 16, 1, D, bounds=True)
        q = torch.ones((1, 2, 1, 1, D), dtype=torch.bfloat16, device="cuda")
        status = ints(0)
        table = torch.arange(9, dtype=torch.int32, device="cuda").reshape(1, 9)
        got = paged_select(q, pages, ints(9*16), table, 3, 0, 1, status=status)
        assert got.tolist() == [[[0, 1, 8]]] and int(status) == BAD_PAGE
        status.zero_()
        lse = torch.zeros((1, 2, 1), device="cuda")
        out = paged_decode(q, pages, ints(9*16), table, got, lse_out=lse, status=status)
        assert bool((out == 0).all()) and bool((lse == -math.inf).all())
        assert int(status) == BAD_PAGE


def test_bounds_hold_every_score():
    """What select ranks by is an upper bound of q.k for the keys of a block."""
    g = gen(14)
    for e4m3 in (False, True):
        cache = PagedKVCache(40, 16, 2, 2, 64, dtype=torch.float16, e4m3=e4m3, bounds=True)
        for n in (100, 1, 1, 30):
            cache.append(randn(g, 2, 2, n, 64).half(), randn(g, 2, 2, n, 64).half())
        k = stored(cache.pages, "k")
        for b in range(2):
            for x in range(-(-132//16)):
                p = int(cache.block_table[b, x])
                rows = k[p, :, :min(16, 132 - 16*x)]
                assert bool((rows.amin(1).half() == cache.pages.bounds[p, :, 0]).all())
                assert bool((rows.amax(1).half() == cache.pages.bounds[p, :, 1]).all())


# ------------------------------------------------------------------------- used together

@pytest.mark.parametrize("e4m3", [False, True])
def test_a_cache_in_use(e4m3):
    """Prompts of different lengths, steps, selected blocks, a sequence that ends and its
    pages going to another: every answer against 64 bits."""
    g = gen(20)
    H, B, D, G, P = 2, 3, 64, 4, 16
    cache = PagedKVCache(60, P, H, B, D, max_blocks=25, dtype=torch.bfloat16, e4m3=e4m3,
                         bounds=True)

    def rows(n):
        return randn(g, H, B, n, D).bfloat16()

    def answer(S=None):
        q = randn(g, H, G, B, 1, D).bfloat16()
        sel = None
        if S:
            sel = paged_select(q, cache.pages, cache.lengths, cache.block_table, S, 1, 1)
            assert torch.equal(sel, chosen(q, cache.pages.bounds, cache.lengths,
                                           cache.block_table, P, S, 1, 1))
        want, _ = check_attention(q, cache.pages, cache.lengths, cache.block_table, sel)
        assert torch.equal(cache.decode(q, num_selected=S), want)

    cache.append(rows(200), rows(200), [200, 31, 90])
    answer()
    for _ in range(3):
        cache.append(rows(1), rows(1))
        answer()
        answer(4)
    cache.release(0)
    answer()
    cache.append(rows(150), rows(150), [150, 0, 2])
    answer()
    answer(3)
    k, v = cache.read()
    assert k.shape == (H, B, 150, D) and bool((k[:, 1, 34:] == 0).all())
    cache.clear()
    assert len(cache) == 0 and cache.free_pages == 60


def test_on_another_stream_and_on_slices_of_larger_buffers():
    """Work goes to the current stream; buffers may start anywhere."""
    g = gen(21)
    H, B, D, P, n = 2, 2, 64, 16, 100
    side = torch.cuda.Stream()
    store = torch.zeros(20*H*P*D*2 + 8, dtype=torch.float16, device="cuda")
    for shift in (0, 1, 8):
        size = 20*H*P*D
        pages = KVPages(store[shift:shift + size].view(20, H, P, D),
                        store[shift + size:shift + 2*size].view(20, H, P, D))
        table = make_table(g, [n, n], P, 20)
        k, v = randn(g, H, B, n, D).half(), randn(g, H, B, n, D).half()
        q = randn(g, H, 3, B, 1, D).half()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            torch.cuda._sleep(2_000_000)                     # the main stream would be too early
            paged_append(pages, ints(0, 0), table, k, v)
            out = paged_decode(q, pages, ints(n, n), table)
        torch.cuda.current_stream().wait_stream(side)
        want, _ = check_attention(q, pages, ints(n, n), table)
        assert torch.equal(out, want)


def test_pages_whose_buffers_are_made_on_access():
    """Attributes of a pool may be computed: what they return lives until the call is made."""
    class Views(KVPages):
        __slots__ = ("whole",)
        k = property(lambda self: self.whole[:1].view(self.whole.shape[1:]))
        v = property(lambda self: self.whole[1:].view(self.whole.shape[1:]))
        k_scales = v_scales = bounds = None
        e4m3 = False

        def __init__(self, whole):
            self.whole = whole

    g = gen(27)
    H, D, P, n = 2, 64, 16, 70
    table = make_table(g, [n, n], P, 20)
    whole = randn(g, 2, 20, H, P, D).bfloat16()
    q = randn(g, H, 3, 2, 1, D).bfloat16()
    for _ in range(20):
        got = paged_decode(q, Views(whole), ints(n, n), table)
        assert torch.equal(got, paged_decode(q, KVPages(whole[0], whole[1]), ints(n, n), table))


def test_two_calls_at_once():
    """Calls on two streams, each with the workspace it allocates, do not disturb each other."""
    g = gen(22)
    H, D, P, n = 4, 128, 16, 4000
    pages = make_pool(g, 600, P, H, D, torch.bfloat16, False, bounds=True)
    table = make_table(g, [n, n], P, 600)
    lens = ints(n, n)
    qs = [randn(g, H, 4, 2, 1, D).bfloat16() for _ in range(2)]
    alone = [(paged_select(q, pages, lens, table, 30), paged_decode(q, pages, lens, table))
             for q in qs]
    streams = [torch.cuda.Stream() for _ in qs]
    torch.cuda.synchronize()
    for _ in range(5):
        got = []
        for q, s in zip(qs, streams):
            with torch.cuda.stream(s):
                got.append((paged_select(q, pages, lens, table, 30),
                            paged_decode(q, pages, lens, table)))
        torch.cuda.synchronize()
        for (a, b), (c, d) in zip(alone, got):
            assert torch.equal(a, c) and torch.equal(b, d)


def test_captured_step_with_other_lengths_and_pages():
    """A decode step in a graph, replayed while lengths, table and rows change underneath; a
    second graph over the same buffers and workspaces in turn."""
    g = gen(23)
    H, B, D, G, P, M = 2, 3, 64, 4, 16, 12
    pages = make_pool(g, 50, P, H, D, torch.bfloat16, True, bounds=True)
    table = torch.full((B, M), -1, dtype=torch.int32, device="cuda")
    lens, after = ints(0, 0, 0), ints(1, 1, 1)
    k, v = (torch.zeros((H, B, 1, D), dtype=torch.bfloat16, device="cuda") for _ in range(2))
    q = torch.zeros((H, G, B, 1, D), dtype=torch.bfloat16, device="cuda")
    sel = torch.empty((H, B, 4), dtype=torch.int32, device="cuda")
    out, dense = torch.empty_like(q), torch.empty_like(q)
    ws = torch.empty(1 << 22, dtype=torch.uint8, device="cuda")
    ws2 = torch.empty(1 << 16, dtype=torch.uint8, device="cuda")

    def step():
        paged_append(pages, lens, table, k, v)
        paged_select(q, pages, after, table, 4, 1, 1, out=sel, workspace=ws2)
        paged_decode(q, pages, after, table, sel, out=out, workspace=ws)

    def whole():
        paged_decode(q, pages, after, table, out=dense, workspace=ws)

    table.copy_(make_table(g, [1, 1, 1], P, 50, spare=M - 1))
    step()
    whole()
    graphs = []
    for f in (step, whole):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            f()
        graphs.append(graph)
    for lengths in ([40, 0, 191], [100, 15, 16], [3, 80, 81]):
        ends = [n + 1 for n in lengths]
        table.copy_(make_table(g, ends, P, 50, spare=M - -(-max(ends)//P)))
        lens.copy_(ints(*lengths))
        after.copy_(ints(*ends))
        kk = stored(pages, "k")
        pages.bounds.copy_(torch.stack([kk.amin(2), kk.amax(2)], 2).bfloat16())
        for t in (k, v, q):
            t.copy_(randn(g, *t.shape))
        for graph in graphs + graphs:
            graph.replay()
        assert torch.equal(sel, chosen(q, pages.bounds, after, table, P, 4, 1, 1))
        assert torch.equal(out, check_attention(q, pages, after, table, sel)[0])
        assert torch.equal(dense, check_attention(q, pages, after, table)[0])


def test_lengths_and_tables_written_just_before_each_call():
    """Every call of a step reads what the kernel right before it in the stream has written
    (lengths by an addition, table, rows and queries by copies), eagerly and in a graph whose
    steps also fork to another stream."""
    g = gen(25)
    H, B, D, G, P, M = 2, 5, 64, 4, 16, 41                   # room for 656 positions
    pages = make_pool(g, B*M, P, H, D, torch.bfloat16, False, bounds=True)
    table = torch.randperm(B*M, generator=g, device="cuda", dtype=torch.int32).reshape(B, M)
    zero = torch.zeros((), dtype=torch.int32, device="cuda")
    real, lens, after, work = ints(300, 17, 620, 0, 95), ints(0, 0, 0, 0, 0), ints(0, 0, 0, 0, 0), \
        torch.zeros_like(table)
    k = randn(g, H, B, 1, D).bfloat16()
    src = randn(g, H, G, B, 1, D).bfloat16()
    q = torch.zeros_like(src)
    out = [torch.zeros_like(src) for _ in range(3)]
    sel = [torch.zeros((H, B, n), dtype=torch.int32, device="cuda") for n in (5, M)]
    side = torch.cuda.Stream()

    def step():
        lens.copy_(real)
        work.copy_(table)
        paged_append(pages, lens, work, k, k)
        torch.add(lens, zero + 1, out=after)
        paged_decode(q, pages, after, work, out=out[0])         # of the queries before
        q.copy_(src)
        paged_select(q, pages, after, work, 5, 1, 1, out=sel[0])
        paged_decode(q, pages, after, work, sel[0], out=out[1])
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            paged_decode(q, pages, after, work, out=out[2])
        after.add_(0)
        paged_select(q, pages, after, work, M, 0, 0, out=sel[1])
        torch.cuda.current_stream().wait_stream(side)
        lens.zero_()
        work.fill_(-1)
        after.zero_()

    def check():
        ends = real + 1
        assert torch.equal(sel[0], chosen(q, pages.bounds, ends, table, P, 5, 1, 1))
        assert torch.equal(sel[1], chosen(q, pages.bounds, ends, table, P, M, 0, 0))
        assert torch.equal(out[1], check_attention(src, pages, ends, table, sel[0])[0])
        assert torch.equal(out[2], check_attention(src, pages, ends, table)[0])

    for _ in range(3):
        step()
    torch.cuda.synchronize()
    check()
    assert torch.equal(out[0], out[2])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
        step()
    for _ in range(3):
        real += 7
        real[3] = 0
        src.copy_(randn(g, *src.shape))
        graph.replay()
        graph.replay()
        check()
        assert torch.equal(out[0], out[2])


def test_offsets_past_32_bits():
    """Pages behind 4 GB of codes, 2^32 elements into the pool."""
    H, P, D = 8, 64, 128
    N = (1 << 32)//(H*P*D) + 40
    g = gen(24)
    pages = KVPages.empty(N, P, H, D, torch.bfloat16, e4m3=True, bounds=True)
    table = (N - 1 - torch.arange(8, device="cuda", dtype=torch.int32)).reshape(1, 8)
    n = 8*P - 3
    k, v = randn(g, H, 1, n, D).bfloat16(), randn(g, H, 1, n, D).bfloat16()
    paged_append(pages, ints(0), table, k, v)
    ko, vo = torch.zeros_like(k), torch.zeros_like(v)
    paged_gather(pages, ints(n), table, ko, vo)
    assert same(ko.double(), quantised(k.double())[0].bfloat16().double())
    assert same(vo.double(), quantised(v.double())[0].bfloat16().double())
    # the same rows in a small pool give the same answers, bit for bit
    small = KVPages.empty(8, P, H, D, torch.bfloat16, e4m3=True, bounds=True)
    near = torch.arange(8, device="cuda", dtype=torch.int32).reshape(1, 8)
    paged_append(small, ints(0), near, k, v)
    q = randn(g, H, 4, 1, 1, D).bfloat16()
    assert torch.equal(paged_select(q, pages, ints(n), table, 4), paged_select(q, small, ints(n), near, 4))
    assert torch.equal(paged_decode(q, pages, ints(n), table), paged_decode(q, small, ints(n), near))


def test_small_workspaces_are_refused():
    pages = KVPages.empty(4, 16, 1, 64, bounds=True)
    q = torch.zeros((1, 1, 1, 1, 64), dtype=torch.bfloat16, device="cuda")
    ws = torch.empty(0, dtype=torch.uint8, device="cuda")
    table = ints(0, 1, 2, 3).reshape(1, 4)
    for call in (lambda: paged_decode(q, pages, ints(9), table, workspace=ws),
                 lambda: paged_select(q, pages, ints(9), table, 1, 1, 0, workspace=ws)):
        with pytest.raises((_lib.StatusError, ValueError)):
            call()
    assert ops.paged_decode_workspace_bytes(64, 16, 4, 1, 1, 1) > 0
