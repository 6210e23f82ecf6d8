"""Values, weights and scores of unusual size through the paged decode, element by element
against 64 bits.

With p_i the softmax weights, s_i the scale of a value row (1 in 16-bit pages), u the half
step of the output's type, ds a score's error, n the number of positions (test_gpu_paged.py
derives ds, the 2^-15 and the n * 2^-23):

  |out_d - exact_d| <= u*|exact_d| + (4 ds + 2^-15 + n * 2^-23) * sum_i p_i |v_id| + tail_d

The tail is there for weights that go through fp16 operands (fp16 rows, 8-bit rows).  A weight
p_i s_i enters with 22 bits and not finer than 2^-24 in units that make the largest of its tile,
rows that are all zero left out, one or more.  So tail_d = 2^-24 * max_j(p_j s_j) * sum_i
|v_id|/s_i, over rows that are not zero; bf16 weights have the exponents of fp32 and no tail.
Everything in the bound is of the same sequence, kv head and query head as the output."""
import math

import pytest
import torch

from nntile_b200.sdpa import KVPages, paged_append, paged_decode
from test_gpu_paged import DT, gen, ints, make_pool, make_table, randn, stored, two_to

pytestmark = pytest.mark.gpu


def exact(q, pages, lengths, table, selected=None):
    """(out, its bound, lse, its bound), 64 bits."""
    H, G, B, _, D = q.shape
    P = pages.k.shape[2]
    K, V = stored(pages, "k"), stored(pages, "v")
    half = torch.finfo(q.dtype).eps/2
    least = torch.finfo(q.dtype).smallest_normal*torch.finfo(q.dtype).eps
    out = torch.zeros((H, G, B, 1, D), dtype=torch.float64, device="cuda")
    tol = torch.zeros_like(out)
    lse = torch.full((H, G, B), -math.inf, dtype=torch.float64, device="cuda")
    lse_tol = torch.zeros_like(lse)
    for b, n in enumerate(lengths.tolist()):
        for h in range(H):
            blocks = list(range(-(-n//P))) if selected is None else \
                [x for x in selected[h, b].tolist() if 0 <= x < -(-n//P)]
            if not blocks:
                continue
            where = [(int(table[b, x]), min(P, n - x*P)) for x in blocks]
            k, v = (torch.cat([T[p, h, :r] for p, r in where]) for T in (K, V))
            s = torch.ones(len(k), dtype=torch.float64, device="cuda")
            if pages.e4m3:
                s = torch.cat([two_to(pages.v_scales[p, h, :r].long() - 127) for p, r in where])
            qq = q[h, :, b, 0].double()
            score = qq @ k.T/math.sqrt(D)
            lse[h, :, b] = torch.logsumexp(score, -1)
            p = torch.softmax(score, -1)
            # position by position: 0 * inf of another position must not get in
            out[h, :, b, 0] = (p[:, :, None]*v[None]).sum(1)
            ds = (D + 16)*2.0**-23/math.sqrt(D)*(qq.abs() @ k.abs().T).amax(-1)
            part = 4*ds + 2.0**-15 + len(k)*2.0**-23
            size = torch.where(v.isfinite(), v, 0.0).abs()
            tail = 0.0
            if pages.e4m3 or q.dtype == torch.float16:
                live = (v != 0).any(-1)
                top = (p*s*live).amax(-1)
                tail = 2.0**-24*top[:, None]*(size/s[:, None]).sum(0)
            tol[h, :, b, 0] = half*out[h, :, b, 0].abs() + part[:, None]*(p @ size) + tail + least
            lse_tol[h, :, b] = 2*ds + 2.0**-21*(1 + lse[h, :, b].abs()) + len(k)*2.0**-23
    return out, tol, lse, lse_tol


def check(q, pages, lengths, table, selected=None):
    want, tol, want_lse, lse_tol = exact(q, pages, lengths, table, selected)
    lse = torch.full(q.shape[:3], math.nan, dtype=torch.float32, device="cuda")
    status = ints(0)
    out = paged_decode(q, pages, lengths, table, selected, lse_out=lse, status=status)
    assert int(status) == 0
    rounded = want.to(q.dtype).double()          # what is past the type's range is infinite
    fine = rounded.isfinite()
    assert bool(((out.double() == rounded) | (out.isnan() & rounded.isnan()))[~fine].all())
    off = (out.double() - want).abs()
    assert bool((off <= tol)[fine].all()), float((off/tol)[fine].nan_to_num(math.inf).max())
    some = want_lse > -math.inf
    assert bool((lse[~some] == -math.inf).all())
    assert bool(((lse.double() - want_lse).abs() <= lse_tol)[some].all())
    assert torch.equal(out.view(torch.int16), paged_decode(q, pages, lengths, table, selected)
                       .view(torch.int16))       # and the same again, bit for bit
    return out


def fill(pages, table, lengths, k, v):
    paged_append(pages, torch.zeros_like(lengths), table, k, v, lengths)


# -------------------------------------------------------------------------- infinite values

@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("D,P,G,n", [
    (128, 16, 4, 1), (64, 16, 1, 1), (256, 16, 2, 1), (128, 16, 9, 1), (80, 16, 3, 1), (20, 5, 2, 1),
    (128, 16, 4, 500), (64, 32, 9, 300), (256, 16, 2, 700), (80, 16, 3, 6000), (128, 16, 1, 20000),
    (20, 5, 2, 300)])
def test_infinite_values_stay_infinite(D, P, G, n, dtype):
    """An infinity in a value row makes its column of the output infinite; two of opposite sign,
    or a NaN, make it NaN; the other columns do not notice."""
    dt, g = DT[dtype], gen(D + n)
    H, lens = 2, [n, max(1, n//3)]
    N = sum(-(-x//P) for x in lens) + 1
    pages = KVPages.empty(N, P, H, D, dt)
    table, lengths = make_table(g, lens, P, N), ints(*lens)
    k, v = randn(g, H, 2, n, D), randn(g, H, 2, n, D)
    v[0, 0, 0, 0] = math.inf
    v[0, 1, lens[1] - 1, 1] = -math.inf
    v[1, 0, n//2, 2], v[1, 0, n - 1, 2] = math.inf, math.inf
    v[1, 0, n//2, 3], v[1, 0, n - 1, 4] = -math.inf, math.nan
    v[1, 1, 0, 5], v[1, 1, lens[1] - 1, 5] = math.inf, (math.inf if n == 1 else -math.inf)
    fill(pages, table, lengths, k.to(dt), v.to(dt))
    q = randn(g, H, G, 2, 1, D).to(dt)
    out = check(q, pages, lengths, table)
    assert bool((out[0, :, 0, 0, 0] == math.inf).all())
    assert bool((out[0, :, 1, 0, 1] == -math.inf).all())
    sel = torch.tensor([0, (n - 1)//P, n//2//P, -1], dtype=torch.int32, device="cuda").unique()
    check(q, pages, lengths, table, sel.expand(H, 2, -1).contiguous())


# ------------------------------------------------------- value rows of very different size

SHAPES = [(64, 16, 1), (64, 32, 9), (128, 16, 4), (128, 64, 12), (256, 16, 2), (80, 16, 3), (96, 16, 9),
          (72, 5, 3)]


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("D,P,G", SHAPES)
@pytest.mark.parametrize("n", [16, 100, 5000])
def test_a_row_of_zeros_that_takes_the_weight(n, D, P, G, e4m3, dtype):
    """One position, first, in the middle or last, has all of the weight and no value: what is
    left of the others is the answer, also when it is very little."""
    dt, g = DT[dtype], gen(n + D + G)
    B = 6
    N = B*(-(-n//P))
    pages = KVPages.empty(N, P, 1, D, dt, e4m3)
    table, lengths = make_table(g, [n]*B, P, N), ints(*[n]*B)
    k, v = 0.02*randn(g, 1, B, n, D), randn(g, 1, B, n, D)
    q = randn(g, 1, G, B, 1, D).to(dt)
    q[..., 0] = 1.0
    k[..., 0] = 0.0
    for b, (at, gap) in enumerate([(0, 8), (0, 14), (n//2, 16), (n - 1, 20), (3, 30), (n//3, 45)]):
        k[:, b, at] = 0.0
        k[:, b, at, 0] = gap*math.sqrt(D)
        v[:, b, at] = 0.0
    # small enough for an 8-bit row of them to have a small scale, large enough for the output
    v *= 0.02 if dtype == "bf16" else 2.0**13
    fill(pages, table, lengths, k.to(dt), v.to(dt))
    check(q, pages, lengths, table)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("D,P,G", SHAPES)
@pytest.mark.parametrize("n", [40, 3000])
def test_large_rows_without_weight(n, D, P, G, e4m3, dtype):
    """Value rows up to 2^60 (bf16) or 2^29 (fp16) larger than the others whose weight is next to
    nothing, at the beginning, the end and in between, several in a sequence."""
    dt, g = DT[dtype], gen(n + D + 2*G)
    apart = [20, 28, 36, 60] if dtype == "bf16" else [16, 22, 29, 29]
    B = len(apart)
    N = B*(-(-n//P))
    pages = KVPages.empty(N, P, 2, D, dt, e4m3)
    table, lengths = make_table(g, [n]*B, P, N), ints(*[n]*B)
    k, v = 0.05*randn(g, 2, B, n, D), randn(g, 2, B, n, D)
    q = randn(g, 2, G, B, 1, D).to(dt)
    q[..., 0] = 1.0
    k[..., 0] = 0.0
    small = 1.0 if dtype == "bf16" else 2.0**-14
    v *= small
    for b, x in enumerate(apart):
        for at in (0, 5, n//2, n - 1):
            v[:, b, at] *= 2.0**x/4
            k[:, b, at, 0] = -(x*0.7 + 10)*math.sqrt(D)
    fill(pages, table, lengths, k.to(dt), v.to(dt))
    check(q, pages, lengths, table)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("D,P,G", SHAPES)
@pytest.mark.parametrize("size", [1.0, 5.0, 12.0])
def test_scores_of_wide_spread(size, D, P, G, e4m3, dtype):
    """Scores over up to a hundred binades and value rows over twelve, rows of zeros among
    them."""
    dt, g = DT[dtype], gen(D + P + G)
    lens = [1, 17, 300, 2100, 0, 33]
    H, n = 2, max(lens)
    N = sum(-(-x//P) for x in lens) + 1
    pages = KVPages.empty(N, P, H, D, dt, e4m3)
    table, lengths = make_table(g, lens, P, N), ints(*lens)
    k, v = randn(g, H, len(lens), n, D), randn(g, H, len(lens), n, D)
    v *= torch.exp2(torch.randint(-6, 7, (H, len(lens), n, 1), generator=g, device="cuda").float())
    v[torch.rand((H, len(lens), n), generator=g, device="cuda") < 0.1] = 0.0
    fill(pages, table, lengths, k.to(dt), v.to(dt))
    check((size*randn(g, H, G, len(lens), 1, D)).to(dt), pages, lengths, table)


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("D,P,G", SHAPES)
@pytest.mark.parametrize("power", [-110, -70, -40, 50, 100])
def test_values_of_any_size(power, D, P, G, e4m3):
    """All of a cache's values are tiny or huge, a row of zeros with half of the weight first."""
    g, lens = gen(D + G - power), [1, 30, 700]
    N = sum(-(-x//P) for x in lens)
    pages = KVPages.empty(N, P, 1, D, torch.bfloat16, e4m3)
    table, lengths = make_table(g, lens, P, N), ints(*lens)
    k, v = randn(g, 1, 3, 700, D), randn(g, 1, 3, 700, D)*2.0**power
    v[:, 2, 0] = 0.0
    k[:, 2, 0, 0] = 5*math.sqrt(D)
    q = randn(g, 1, G, 3, 1, D)
    q[..., 0] = 1.0
    fill(pages, table, lengths, k.bfloat16(), v.bfloat16())
    check(q.bfloat16(), pages, lengths, table)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("D,P,G", SHAPES)
def test_rows_that_grow_as_their_weights_shrink(D, P, G, e4m3, dtype):
    """Rows over 70 binades (fp16: 26) along the sequence, up and down, with weights that make
    all of them count the same, or only the small ones."""
    dt, g = DT[dtype], gen(D + 3*G)
    n, span = 1500, 70 if dtype == "bf16" else 26
    N = 4*(-(-n//P))
    pages = KVPages.empty(N, P, 1, D, dt, e4m3)
    table, lengths = make_table(g, [n]*4, P, N), ints(*[n]*4)
    k, v = 0.1*randn(g, 1, 4, n, D), randn(g, 1, 4, n, D)
    binades = torch.arange(n, device="cuda")/n*span - span/2
    for b, (x, y) in enumerate([(binades, 1.0), (-binades, 1.0), (binades, 1.6), (-binades, 1.6)]):
        v[0, b] *= torch.exp2(x.round())[:, None]
        k[0, b, :, 0] = -y*x*math.log(2)*math.sqrt(D)
    q = 0.1*randn(g, 1, G, 4, 1, D)
    q[..., 0] = 1.0
    fill(pages, table, lengths, k.to(dt), v.to(dt))
    check(q.to(dt), pages, lengths, table)


@pytest.mark.parametrize("e4m3", [False, True])
def test_scores_that_rise_fall_and_rise(e4m3):
    """The largest scores of a tile climb and sink by hundreds of binades along the sequence."""
    g = gen(40)
    D, P, G, n = 64, 16, 4, 4000
    for dt in DT.values():
        pages = KVPages.empty(n//P, P, 1, D, dt, e4m3)
        table, lengths = make_table(g, [n], P, n//P), ints(n)
        k, v = 0.1*randn(g, 1, 1, n, D), randn(g, 1, 1, n, D)
        at = torch.arange(n, device="cuda")
        k[..., 0] = 8*(100*torch.sin(at/300.0) + 20*torch.sin(at/37.0))
        q = randn(g, 1, G, 1, 1, D)
        q[..., 0] = torch.tensor([1.0, -1.0, 0.25, 0.0], device="cuda")[:, None, None]
        fill(pages, table, lengths, k.to(dt), v.to(dt))
        check(q.to(dt), pages, lengths, table)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("D,P,G,lens", [(64, 16, 1, [1, 5, 130]), (128, 64, 8, [65, 700]), (256, 16, 2, [35]),
                                        (96, 32, 12, [33, 1000])])
def test_scales_behind_a_sequence_hold_anything(D, P, G, lens, dtype):
    dt, g = DT[dtype], gen(D + 7)
    N = sum(-(-x//P) for x in lens) + 2
    pages = make_pool(g, N, P, 2, D, dt, True)
    table, lengths = make_table(g, lens, P, N), ints(*lens)
    q = randn(g, 2, G, len(lens), 1, D).to(dt)
    live = torch.zeros((N, P), dtype=torch.bool, device="cuda")
    for b, x in enumerate(lens):
        for i in range(x):
            live[int(table[b, i//P]), i % P] = True
    want = check(q, pages, lengths, table)
    for byte in (0, 1, 254, 255):
        for t in (pages.k_scales, pages.v_scales):
            t.masked_fill_(~live[:, None], byte)
        assert torch.equal(paged_decode(q, pages, lengths, table), want)
    for t in (pages.k, pages.v):
        t.masked_fill_(~live[:, None, :, None], 0x7F)
    assert torch.equal(paged_decode(q, pages, lengths, table), want)
