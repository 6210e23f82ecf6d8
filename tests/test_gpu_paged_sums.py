"""Sums over long sequences through the paged decode are fp32 sums that round to nearest.

All scores are one of two numbers, the larger at the first position of a page, so that weights are
two fp32 numbers of many bits, and the output is a mean of the values in which a weight's own
error, the same for 63 of 64 positions, all but cancels.  What is off is the sum alone.  A share of
the sequence here has T = 2048 tiles, and their sums are added one after the other.  Rounded to
nearest, each addition is off by a random part of half a step, 2^-25 of the sum in the mean square
and less; six standard deviations of T of them are 6 * sqrt(2048) * 2^-25 < 8.1e-6 of the sum (cut
off instead, T * 2^-25 on one side: 6.1e-5).  An output then differs from the exact mean rounded to
its type where that mean is this near to the middle of two numbers: 8.1e-6 * 1.5 out of a step,
which is 2^-10 (fp16) or 2^-7 (bf16) for means in [1, 1.5], so 1.25 % and 0.16 % of outputs that
lie anywhere in a step.  The test allows as many, and six standard deviations of that count.  The
kernel for other pages adds up fewer sums, of 64 positions each."""
import math

import pytest
import torch

from nntile_b200.sdpa import KVPages, paged_append, paged_decode
from test_gpu_paged import DT, gen, ints

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("D,G,P", [(64, 1, 64), (128, 9, 64),
                                   (64, 1, 40), (128, 9, 40)])      # without the tensor instruction
def test_means_of_long_sequences(D, G, P, e4m3, dtype):
    dt, g = DT[dtype], gen(D)
    H, B, own, blocks = 8, 37, 16, 131072//P                 # 296 units of 131072 positions
    pages = KVPages.empty(B*own, P, H, D, dt, e4m3)
    # values of 1 and 1.5, in parts that differ by sequence, head and column
    part = torch.rand((H, B, 1, D), generator=g, device="cuda")
    v = 1.0 + 0.5*(torch.rand((H, B, own*P, D), generator=g, device="cuda") < part).float()
    table = torch.arange(B*own, dtype=torch.int32, device="cuda").reshape(B, own)
    k = torch.zeros_like(v)
    k[..., 0] = 1.0
    k[:, :, ::P, 0] = 2.0
    paged_append(pages, ints(*[0]*B), table, k.to(dt), v.to(dt))
    # every page of a sequence many times, as a read may
    pick = torch.randint(0, own, (B, blocks), generator=g, device="cuda")
    long = torch.gather(table, 1, pick).contiguous()
    many = torch.zeros((B, own), dtype=torch.float64, device="cuda")
    many.scatter_add_(1, pick, torch.ones_like(pick, dtype=torch.float64))
    weight = torch.softmax(k[0, 0, :P, 0].double()/math.sqrt(D), 0)
    mean = torch.einsum("hbprd,bp,r->hbd", v.double().reshape(H, B, own, P, D), many, weight)/blocks
    q = torch.zeros((H, G, B, 1, D), dtype=dt, device="cuda")
    q[..., 0] = 1.0
    out = paged_decode(q, pages, ints(*[blocks*P]*B), long)
    assert bool((out == out[:, :1]).all())
    wrong = float((out[:, 0, :, 0] != mean.to(dt)).double().mean())
    step = torch.finfo(dt).eps
    allowed = 6*math.sqrt(2048)*2.0**-25*1.5/step
    assert wrong <= allowed + 6*math.sqrt(allowed/mean.numel()), (wrong, allowed)
    assert float((out[:, 0, :, 0].double() - mean).abs().max()) <= step*0.5 + 2048*2.0**-24*1.5
