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
from test_gpu_paged import DT, gen, ints, make_table, randn, stored, two_to

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
