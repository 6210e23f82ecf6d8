"""What the paged key-value cache operators are measured on.

Cases stand for what a serving program does with such a cache: it writes the new rows of every
sequence into pages, reads pages back for a prompt's next part, answers one new token per sequence
from all of a cache, or from those blocks of it that a cheap score picks.

Arrays are contiguous torch tensors in the framework's (reversed Fortran) order:
q (kv_heads, group, batch, 1, head); k, v of new rows (kv_heads, batch, rows, head);
pages (num_pages, kv_heads, page, head); scales of 8-bit pages (num_pages, kv_heads, page), an
exponent byte e each: value = code * 2**(e - 127); bounds (num_pages, kv_heads, 2, head), the least
and the largest stored key of a page; block_table (batch, max_blocks); lengths (batch).
"""
import math
import random

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def listed():
    return [
        # one new row for each sequence of a batch, pages with bounds: every step of a decode loop
        {"name": "append_step_bf16", "kind": "append", "dtype": "bf16", "e4m3": False, "head": 128, "page": 16,
         "kv_heads": 8, "group": 4, "batch": 64, "length": 1000, "new": 1, "selected": 0, "mix": 1},
        # a batch of prompts written at once, ragged
        {"name": "append_prompt_fp16", "kind": "append", "dtype": "fp16", "e4m3": False, "head": 128, "page": 32,
         "kv_heads": 8, "group": 4, "batch": 4, "length": 45, "new": 4096, "selected": 0, "mix": 2},
        # a prompt's part goes into an 8-bit cache and the whole cache is read back for its attention
        {"name": "store_and_read_e4m3", "kind": "store", "dtype": "bf16", "e4m3": True, "head": 128, "page": 64,
         "kv_heads": 8, "group": 4, "batch": 8, "length": 5001, "new": 1023, "selected": 0, "mix": 3},
        # a 12-head cache of short sequences read back
        {"name": "read_e4m3_head64", "kind": "read", "dtype": "fp16", "e4m3": True, "head": 64, "page": 16,
         "kv_heads": 12, "group": 1, "batch": 3, "length": 333, "new": 0, "selected": 0, "mix": 4},
        # pages of the rows' own type read back, long
        {"name": "read_bf16", "kind": "read", "dtype": "bf16", "e4m3": False, "head": 128, "page": 16,
         "kv_heads": 8, "group": 4, "batch": 16, "length": 8192, "new": 0, "selected": 0, "mix": 5},
        # one user's first answers: latency
        {"name": "decode_short_bf16", "kind": "decode", "dtype": "bf16", "e4m3": False, "head": 64, "page": 16,
         "kv_heads": 12, "group": 1, "batch": 1, "length": 129, "new": 0, "selected": 0, "mix": 0},
        # the decode workload of the benchmark, in pages: 64 sequences of 8192
        {"name": "decode_full_bf16", "kind": "decode", "dtype": "bf16", "e4m3": False, "head": 128, "page": 16,
         "kv_heads": 8, "group": 4, "batch": 64, "length": 8192, "new": 0, "selected": 0, "mix": 0},
        # a served batch of very different lengths in 8 bits, one slot of it empty
        {"name": "decode_ragged_e4m3", "kind": "decode", "dtype": "bf16", "e4m3": True, "head": 128, "page": 64,
         "kv_heads": 8, "group": 8, "batch": 37, "length": 16383, "new": 0, "selected": 0, "mix": 6},
        # one long document, few key heads: the split over the length decides
        {"name": "decode_long_fp16", "kind": "decode", "dtype": "fp16", "e4m3": False, "head": 128, "page": 32,
         "kv_heads": 2, "group": 7, "batch": 1, "length": 100003, "new": 0, "selected": 0, "mix": 0},
        # blocks of long sequences scored and selected
        {"name": "select_bf16", "kind": "select", "dtype": "bf16", "e4m3": False, "head": 128, "page": 16,
         "kv_heads": 8, "group": 4, "batch": 24, "length": 32769, "new": 0, "selected": 128, "mix": 7},
        # the same with the attention over the blocks, one long sequence
        {"name": "sparse_long_bf16", "kind": "sparse", "dtype": "bf16", "e4m3": False, "head": 128, "page": 32,
         "kv_heads": 8, "group": 4, "batch": 1, "length": 131072, "new": 0, "selected": 64, "mix": 0},
        # and for a ragged batch in 8 bits
        {"name": "sparse_ragged_e4m3", "kind": "sparse", "dtype": "fp16", "e4m3": True, "head": 128, "page": 64,
         "kv_heads": 4, "group": 8, "batch": 29, "length": 20000, "new": 0, "selected": 33, "mix": 8},
    ]


def spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["append", "store", "read", "decode", "decode", "decode", "select", "sparse", "sparse"])
    case = {"kind": kind, "dtype": rng.choice(["bf16", "fp16"]), "e4m3": kind == "store",
            "head": rng.choice([64, 64, 80, 96, 128, 128, 128, 256]), "page": rng.choice([16, 32, 64, 128]),
            "kv_heads": rng.randint(1, 12), "group": rng.randint(1, 9), "batch": spread(rng, 1, 64),
            "length": spread(rng, 1, 120000), "new": 0, "selected": 0, "mix": rng.randint(0, 1 << 20)}
    if kind in ("read", "decode", "sparse"):
        case["e4m3"] = rng.random() < 0.5
    if kind in ("append", "store"):
        case["length"], case["new"] = rng.randint(0, 6000), spread(rng, 1, 4096)
    if kind in ("select", "sparse"):
        case["page"], case["selected"] = rng.choice([16, 32, 64]), spread(rng, 3, 150)
        case["length"] = max(case["length"], 2 * case["page"] * case["selected"])    # something is left out
        case["batch"] = min(case["batch"], (1 << 28) // (case["length"] * case["kv_heads"] * case["head"]) + 1)
    # a cache of at most about a gigabyte
    row = case["batch"] * case["kv_heads"] * case["head"] * 4
    most = max(1, (1 << 30) // row)
    case["length"], case["new"] = min(case["length"], most), min(case["new"], most)
    return case


def lengths_of(case):
    """Filled positions of every sequence; 'mix' 0 gives all the same, otherwise they differ and one slot may be empty."""
    rng, n = random.Random(case["mix"]), case["length"]
    if case["mix"] == 0 or n == 0:
        return [n] * case["batch"]
    some = [rng.randint(max(1, n // 8), n) for _ in range(case["batch"])]
    return [n] + [0 if case["batch"] >= 8 and k == case["batch"] // 2 else v for k, v in enumerate(some)][1:]


def new_of(case):
    """New rows of every sequence."""
    rng, n = random.Random(case["mix"] + 1), case["new"]
    if case["mix"] == 0 or n <= 1:
        return [n] * case["batch"]
    return [n] + [rng.randint(max(1, n // 4), n) for _ in range(case["batch"] - 1)]


def blocks_of(case):
    return [-(-v // case["page"]) for v in lengths_of(case)]


def filled_of(case):
    return [a + b for a, b in zip(lengths_of(case), new_of(case))]


def forced(case):
    """Blocks at the beginning and at the end of a sequence that are always selected."""
    return (1, 2) if case["selected"] >= 3 else (0, 0)


def two_to(power):
    """2**power in 32 bits, by its bits."""
    return ((power.int() + 127) << 23).view(torch.float32)


def quantised(x):
    """Rows of 32-bit numbers as e4m3 codes and exponent bytes: the least power of two that brings a row's largest size to 448 or less."""
    size = torch.where(x.isfinite(), x, 0.0).abs().amax(-1)
    part, power = torch.frexp(size)
    power = torch.where(part > 0.875, power - 8, power - 9).clamp(-126, 127)
    power = torch.where(size == 0, 0, power)
    scaled = x * two_to(-power)[..., None]
    codes = torch.where(x.isfinite(), scaled, float("nan")).to(torch.float8_e4m3fn)
    return codes.view(torch.uint8), (power + 127).to(torch.uint8)


def values(codes, scales):
    """What pages stand for, in 32 bits."""
    if scales is None:
        return codes.float()
    return codes.view(torch.float8_e4m3fn).float() * two_to(scales.int() - 127)[..., None]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype, page, head, heads, batch = TYPES[case["dtype"]], case["page"], case["head"], case["kv_heads"], case["batch"]

    def normal(*shape):
        return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32 if case["e4m3"] else dtype)

    filled = filled_of(case)
    blocks = [-(-v // page) for v in filled]
    wide = max(1, max(blocks))
    pages = sum(blocks) + 3
    order = torch.randperm(pages, generator=gen, device="cuda", dtype=torch.int32)
    table = torch.full((batch, wide), -1, dtype=torch.int32, device="cuda")
    live = torch.arange(wide, device="cuda")[None, :] < torch.tensor(blocks, device="cuda")[:, None]
    table[live] = order[:sum(blocks)]
    s = {"case": case, "dtype": dtype, "block_table": table,
         "lengths": torch.tensor(lengths_of(case), dtype=torch.int32, device="cuda"),
         "k_scales": None, "v_scales": None, "bounds": None}
    keys = normal(pages, heads, page, head)
    if case["kind"] in ("select", "sparse"):
        keys += 0.5 * normal(pages, heads, 1, head)      # neighbours are alike: some blocks matter more
    vals = normal(pages, heads, page, head)
    if case["e4m3"]:
        (s["k_pages"], s["k_scales"]), (s["v_pages"], s["v_scales"]) = quantised(keys), quantised(vals)
    else:
        s["k_pages"], s["v_pages"] = keys, vals
    if case["kind"] in ("select", "sparse", "append"):
        stored = values(s["k_pages"], s["k_scales"])
        s["bounds"] = torch.stack([stored.amin(2), stored.amax(2)], 2).to(dtype)
    if case["kind"] in ("append", "store"):
        s["new_lens"] = torch.tensor(new_of(case), dtype=torch.int32, device="cuda")
        s["k"] = torch.randn((heads, batch, case["new"], head), generator=gen, device="cuda").to(dtype)
        s["v"] = torch.randn((heads, batch, case["new"], head), generator=gen, device="cuda").to(dtype)
    if case["kind"] in ("read", "store"):
        s["filled"] = torch.tensor(filled, dtype=torch.int32, device="cuda")
        s["k_out"] = torch.zeros((heads, batch, max(filled), head), dtype=dtype, device="cuda")
        s["v_out"] = torch.zeros_like(s["k_out"])
    if case["kind"] in ("decode", "select", "sparse"):
        s["q"] = torch.randn((heads, case["group"], batch, 1, head), generator=gen, device="cuda").to(dtype)
    return s


# ---- the plain forms ----------------------------------------------------------------------------------------

def places(s, first, count, rows):
    """For the rows i < count[b] at positions first[b] + i: which (batch, row) they are, their page and the place in it."""
    page = s["case"]["page"]
    i = torch.arange(rows, device="cuda")[None, :]
    b, i = torch.nonzero(i < count[:, None], as_tuple=True)
    at = first[b].long() + i
    return b, i, s["block_table"][b, at // page].long(), at % page


def plain_append(s):
    b, i, page, off = places(s, s["lengths"], s["new_lens"], s["k"].shape[2])
    k, v = s["k"][:, b, i].transpose(0, 1), s["v"][:, b, i].transpose(0, 1)    # (rows, heads, head)
    if s["case"]["e4m3"]:
        s["k_pages"][page, :, off], s["k_scales"][page, :, off] = quantised(k.float())
        s["v_pages"][page, :, off], s["v_scales"][page, :, off] = quantised(v.float())
    else:
        s["k_pages"][page, :, off], s["v_pages"][page, :, off] = k, v
    if s["bounds"] is not None:
        size = s["case"]["page"]
        blocks = torch.arange(s["block_table"].shape[1], device="cuda")[None, :] * size
        start, end = s["lengths"][:, None], (s["lengths"] + s["new_lens"])[:, None]
        b, n = torch.nonzero((blocks < end) & (blocks + size > start) & (end > start), as_tuple=True)
        where = s["block_table"][b, n].long()
        stored = values(s["k_pages"][where], None if s["k_scales"] is None else s["k_scales"][where])
        at = n[:, None] * size + torch.arange(size, device="cuda")[None, :]
        fresh = ((at >= start[b]) & (at < end[b]))[:, None, :, None]
        old = (n * size < start[b, 0])[:, None, None]
        least = torch.where(fresh, stored, math.inf).amin(2)
        most = torch.where(fresh, stored, -math.inf).amax(2)
        had = s["bounds"][where].float()
        least = torch.where(old, torch.minimum(least, had[:, :, 0]), least)
        most = torch.where(old, torch.maximum(most, had[:, :, 1]), most)
        s["bounds"][where] = torch.stack([least, most], 2).to(s["dtype"])


def plain_read(s):
    b, i, page, off = places(s, torch.zeros_like(s["filled"]), s["filled"], s["k_out"].shape[2])
    ks = None if s["k_scales"] is None else s["k_scales"][page, :, off]
    vs = None if s["v_scales"] is None else s["v_scales"][page, :, off]
    s["k_out"][:, b, i] = values(s["k_pages"][page, :, off], ks).to(s["dtype"]).transpose(0, 1)
    s["v_out"][:, b, i] = values(s["v_pages"][page, :, off], vs).to(s["dtype"]).transpose(0, 1)


def plain_select(s):
    case = s["case"]
    first, last = forced(case)
    count = (s["lengths"].long() + case["page"] - 1) // case["page"]
    bounds = s["bounds"][s["block_table"].long().clamp(min=0)].double()              # (batch, blocks, heads, 2, head)
    q = s["q"][:, :, :, 0].permute(2, 0, 1, 3).double()                              # (batch, heads, group, head)
    score = torch.matmul(q.clamp(min=0), bounds[:, :, :, 1].permute(0, 2, 3, 1)) \
        + torch.matmul(q.clamp(max=0), bounds[:, :, :, 0].permute(0, 2, 3, 1))
    score = score.amax(2).transpose(0, 1)                                            # (heads, batch, blocks)
    n = torch.arange(score.shape[-1], device="cuda")[None, None, :]
    count = count[None, :, None]
    score = torch.where((n < first) | (n >= count - last), math.inf, score)
    score = torch.where(n < count, score, -math.inf)
    best = torch.sort(score, dim=-1, descending=True, stable=True).indices[..., :case["selected"]]
    best = torch.where(best < count, best, score.shape[-1]).sort(-1).values
    best = torch.where(best < score.shape[-1], best, -1).int()
    return torch.nn.functional.pad(best, (0, case["selected"] - best.shape[-1]), value=-1)


def plain_attention(s, selected=None):
    case, page = s["case"], s["case"]["page"]
    heads, group, batch, _, head = s["q"].shape
    if selected is None:
        selected = torch.arange(s["block_table"].shape[1], device="cuda").expand(heads, batch, -1)
    n = selected.long()
    b = torch.arange(batch, device="cuda")[None, :, None]
    where = s["block_table"][b, n.clamp(min=0)].long().clamp(min=0)
    h = torch.arange(heads, device="cuda")[:, None, None]
    ks, vs = (None if x is None else x[where, h] for x in (s["k_scales"], s["v_scales"]))
    k = values(s["k_pages"][where, h], ks).reshape(heads, batch, -1, head)
    v = values(s["v_pages"][where, h], vs).reshape(heads, batch, -1, head)
    at = n[..., None] * page + torch.arange(page, device="cuda")
    live = ((n[..., None] >= 0) & (at < s["lengths"][None, :, None, None])).reshape(heads, batch, 1, -1)
    q = s["q"][:, :, :, 0].transpose(1, 2).float()                                   # (heads, batch, group, head)
    score = torch.matmul(q, k.transpose(2, 3)) / math.sqrt(head)
    score = torch.where(live, score, -math.inf)
    top = score.amax(-1, keepdim=True)
    part = torch.where(live, torch.exp(score - top), 0.0)
    total = part.sum(-1, keepdim=True)
    out = torch.where(total > 0, torch.matmul(part, v) / total, 0.0).to(s["dtype"])
    lse = torch.where(total > 0, top + torch.log(total), -math.inf)
    return out.transpose(1, 2)[:, :, :, None], lse[..., 0].transpose(1, 2)


def run(state):
    s, case = state, state["case"]
    kind = case["kind"]
    if own:
        from nntile_b200 import sdpa
        pages = sdpa.KVPages(s["k_pages"], s["v_pages"], s["k_scales"], s["v_scales"], s["bounds"])
        if kind in ("append", "store"):
            sdpa.paged_append(pages, s["lengths"], s["block_table"], s["k"], s["v"], s["new_lens"])
        if kind in ("read", "store"):
            sdpa.paged_gather(pages, s["filled"], s["block_table"], s["k_out"], s["v_out"])
        if kind in ("select", "sparse"):
            first, last = forced(case)
            selected = sdpa.paged_select(s["q"], pages, s["lengths"], s["block_table"], case["selected"], first, last)
        if kind in ("decode", "sparse"):
            lse = torch.empty(s["q"].shape[:3], dtype=torch.float32, device="cuda")
            out = sdpa.paged_decode(s["q"], pages, s["lengths"], s["block_table"],
                                    selected if kind == "sparse" else None, lse_out=lse)
    else:
        if kind in ("append", "store"):
            plain_append(s)
        if kind in ("read", "store"):
            plain_read(s)
        if kind in ("select", "sparse"):
            selected = plain_select(s)
        if kind in ("decode", "sparse"):
            out, lse = plain_attention(s, selected if kind == "sparse" else None)
    if kind == "append":
        return {"k_pages": s["k_pages"], "v_pages": s["v_pages"], "bounds": s["bounds"]}
    if kind in ("read", "store"):
        return {"k": s["k_out"], "v": s["v_out"]}
    if kind == "select":
        return {"selected": selected}
    if kind == "decode":
        return {"out": out, "lse": lse}
    return {"selected": selected, "out": out, "lse": lse}


def work(case):
    heads, head, page, group, batch = case["kv_heads"], case["head"], case["page"], case["group"], case["batch"]
    row = head + 1 if case["e4m3"] else 2 * head
    kind, total, flops = case["kind"], 0, 0
    if kind in ("append", "store"):
        total += 2 * sum(new_of(case)) * heads * (2 * head + row)
        if kind == "append":                         # the bounds of the touched pages
            touched = [-(-(a + n) // page) - a // page for a, n in zip(lengths_of(case), new_of(case)) if n]
            total += sum(touched) * heads * 4 * head
            flops += 2 * sum(new_of(case)) * heads * head
    if kind in ("read", "store"):
        total += 2 * sum(filled_of(case)) * heads * (2 * head + row)
    if kind in ("select", "sparse"):
        total += sum(blocks_of(case)) * (4 * head * heads + 4) + heads * batch * (2 * group * head + 4 * case["selected"])
        flops += 4 * head * group * heads * sum(blocks_of(case))
    if kind in ("decode", "sparse"):
        tokens = sum(lengths_of(case))
        if kind == "sparse":
            tokens = sum(min(v, case["selected"] * page) for v in lengths_of(case))
        total += 2 * tokens * heads * row + heads * group * batch * (4 * head + 4)
        flops += 4 * head * group * heads * tokens
    return {"bytes": total, "flops": max(1, flops)}


# ---- the definition in 64 bits -------------------------------------------------------------------------------

def exact_power(e):
    return ((e.long() + 1023) << 52).view(torch.float64)


def exact_e4m3(codes, exponents):
    """The numbers that bytes stand for, from the format: a sign, four bits of exponent with bias 7, three of fraction, no infinity."""
    c = codes.long()
    e, m = (c >> 3) & 15, (c & 7).double()
    size = torch.where(e == 0, m * 2.0 ** -9, (8 + m) * exact_power(e - 10))
    size = torch.where((c & 127) == 127, math.nan, size)
    return torch.where(c >= 128, -size, size) * exact_power(exponents.long() - 127)[..., None]


def exact_rounded(x):
    """Rows as an 8-bit cache holds them: x / 2**e to the nearest of its numbers, ties to even, and e."""
    size = x.abs().amax(-1)
    e = torch.ceil(torch.log2(torch.where(size > 0, size, 448.0) / 448.0)).clamp(-126, 127)
    e = torch.where(size * exact_power(-e) > 448.0, e + 1, e)
    e = torch.where((size > 0) & (size * exact_power(1 - e) <= 448.0) & (e > -126), e - 1, e)
    y = x * exact_power(-e)[..., None]
    grain = exact_power(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(y / grain) * grain * exact_power(e)[..., None]


def exact_pages(s, name, which):
    if s[name + "_scales"] is None:
        return s[name + "_pages"][which].double()
    return exact_e4m3(s[name + "_pages"][which], s[name + "_scales"][which])


def exact_sequence(s, name, b, count):
    """The first `count` rows of sequence b: (heads, count, head)."""
    page = s["case"]["page"]
    which = s["block_table"][b, :-(-count // page)].long()
    rows = exact_pages(s, name, which).transpose(0, 1)
    return rows.reshape(rows.shape[0], -1, rows.shape[-1])[:, :count]


def exact(case, seed):
    s = prepare(case, seed)
    kind, page, heads, head, group = case["kind"], case["page"], case["kv_heads"], case["head"], case["group"]
    lengths, new, filled = lengths_of(case), new_of(case), filled_of(case)
    if kind in ("append", "store"):
        pools = {"k": exact_pages(s, "k", slice(None)), "v": exact_pages(s, "v", slice(None))}
        bounds = None if s["bounds"] is None else s["bounds"].double()
        for b in range(case["batch"]):
            at = torch.arange(lengths[b], filled[b], device="cuda")
            where = s["block_table"][b].long()[at // page]
            for name in ("k", "v"):
                rows = s[name][:, b, :new[b]].double()
                pools[name][where, :, at % page] = (exact_rounded(rows) if case["e4m3"] else rows).transpose(0, 1)
            for n in range(lengths[b] // page, -(-filled[b] // page) if new[b] and bounds is not None else 0):
                low, high = max(lengths[b], n * page) - n * page, min(filled[b], (n + 1) * page) - n * page
                p = int(s["block_table"][b, n])
                fresh = pools["k"][p, :, low:high]
                small, large = fresh.min(1).values, fresh.max(1).values
                if low > 0:
                    small, large = torch.minimum(small, bounds[p, :, 0]), torch.maximum(large, bounds[p, :, 1])
                bounds[p, :, 0], bounds[p, :, 1] = small, large
        if kind == "append":
            return {"k_pages": pools["k"], "v_pages": pools["v"], "bounds": bounds}
        for name in ("k", "v"):
            out = torch.zeros_like(s[name + "_out"], dtype=torch.float64)
            for b in range(case["batch"]):
                which = s["block_table"][b, :-(-filled[b] // page)].long()
                out[:, b, :filled[b]] = pools[name][which].transpose(0, 1).reshape(heads, -1, head)[:, :filled[b]]
            pools[name] = out
        return pools
    if kind == "read":
        out = {name: torch.zeros_like(s[name + "_out"], dtype=torch.float64) for name in ("k", "v")}
        for b in range(case["batch"]):
            for name in ("k", "v"):
                out[name][:, b, :filled[b]] = exact_sequence(s, name, b, filled[b])
        return out
    q = s["q"][:, :, :, 0].double()
    result, selected, (first, last) = {}, None, forced(case)
    if kind in ("select", "sparse"):
        selected = torch.full((heads, case["batch"], case["selected"]), -1, dtype=torch.int32, device="cuda")
        for b in range(case["batch"]):
            count = -(-lengths[b] // page)
            if count == 0:
                continue
            bounds = s["bounds"][s["block_table"][b, :count].long()].double()
            best = torch.full((heads, count), -math.inf, dtype=torch.float64, device="cuda")
            for g in range(group):
                high = torch.maximum(q[None, :, g, b] * bounds[:, :, 0], q[None, :, g, b] * bounds[:, :, 1]).sum(-1)
                best = torch.maximum(best, high.T)
            best[:, :first] = math.inf
            best[:, max(0, count - last):] = math.inf
            for h in range(heads):
                order = sorted(range(count), key=best[h].tolist().__getitem__, reverse=True)[:case["selected"]]
                selected[h, b, :len(order)] = torch.tensor(sorted(order), dtype=torch.int32)
        result["selected"] = selected
    if kind == "select":
        return result
    out = torch.zeros_like(s["q"], dtype=torch.float64)
    lse = torch.full(s["q"].shape[:3], -math.inf, dtype=torch.float64, device="cuda")
    for b in range(case["batch"]):
        if lengths[b] == 0:
            continue
        k, v = exact_sequence(s, "k", b, lengths[b]), exact_sequence(s, "v", b, lengths[b])
        score = torch.einsum("hgd,hld->hgl", q[:, :, b], k) / math.sqrt(head)
        if selected is not None:
            chosen = torch.zeros((heads, -(-lengths[b] // page) + 1), dtype=torch.bool, device="cuda")
            chosen.scatter_(1, selected[:, b].long() % chosen.shape[1], True)        # -1 falls on the spare last column
            rows = chosen[:, :-1].repeat_interleave(page, 1)[:, :lengths[b]]
            score = score.masked_fill(~rows[:, None], -math.inf)
        lse[:, :, b] = torch.logsumexp(score, -1)
        out[:, :, b, 0] = torch.einsum("hgl,hld->hgd", torch.softmax(score, -1), v)
    return {**result, "out": out, "lse": lse}
