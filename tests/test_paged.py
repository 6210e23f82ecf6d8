"""Paged key/value cache, what can be checked without a GPU: refusals of the C entry
points, the checks of the Python functions, and the index arithmetic of the kernels on
values that a caller may have left in device memory."""
import ctypes
import os
import shutil
import subprocess

import pytest
import torch

from nntile_b200 import _lib, build, sdpa

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
NULL = ctypes.c_void_p(0)
# an address that is never dereferenced: every call below is refused before a launch
FAKE = ctypes.c_void_p(1 << 20)
ODD = ctypes.c_void_p((1 << 20) + 1)


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(_lib.LIB_PATH):
        build.build()
    return _lib.load()


def test_index_arithmetic_of_the_kernels(tmp_path):
    if shutil.which("g++") is None:
        pytest.skip("no g++")
    exe = str(tmp_path / "paged_check")
    subprocess.run(["g++", "-std=c++17", "-Wall", "-o", exe,
                    os.path.join(ROOT, "tests", "paged_check.cc")], check=True)
    assert subprocess.run([exe]).returncode == 0


def append(lib, sfx="bf16", head=64, page=16, pages=8, blocks=4, batch=2, heads=2, new=1, fmt=0,
           lengths=FAKE, table=FAKE, k=FAKE, v=FAKE, kp=FAKE, vp=FAKE, ks=NULL, vs=NULL, bd=NULL,
           status=NULL):
    return getattr(lib, f"nntile_b200_paged_kv_append_{sfx}")(
        NULL, head, page, pages, blocks, batch, heads, new, fmt, lengths, NULL, table, k, v, kp,
        vp, ks, vs, bd, status)


def gather(lib, sfx="bf16", head=64, page=16, pages=8, blocks=4, batch=2, heads=2, seq=9, fmt=0,
           lengths=FAKE, table=FAKE, kp=FAKE, vp=FAKE, ks=NULL, vs=NULL, k=FAKE, v=FAKE):
    return getattr(lib, f"nntile_b200_paged_kv_gather_{sfx}")(
        NULL, head, page, pages, blocks, batch, heads, seq, fmt, lengths, table, kp, vp, ks, vs,
        k, v, NULL)


def decode(lib, sfx="bf16", head=64, page=16, pages=8, blocks=4, batch=2, group=2, heads=2, sel=0,
           fmt=0, lengths=FAKE, table=FAKE, selected=NULL, q=FAKE, kp=FAKE, vp=FAKE, ks=NULL,
           vs=NULL, out=FAKE, ws=FAKE, ws_bytes=1 << 30):
    return getattr(lib, f"nntile_b200_paged_decode_sdpa_{sfx}")(
        NULL, head, page, pages, blocks, batch, group, heads, sel, fmt, lengths, table, selected,
        q, kp, vp, ks, vs, out, NULL, ws, ws_bytes, NULL)


def select(lib, sfx="bf16", head=64, page=16, pages=8, blocks=4, batch=2, group=2, heads=2, sel=2,
           first=1, last=1, lengths=FAKE, table=FAKE, q=FAKE, bd=FAKE, out=FAKE, ws=FAKE,
           ws_bytes=1 << 30):
    return getattr(lib, f"nntile_b200_paged_select_{sfx}")(
        NULL, head, page, pages, blocks, batch, group, heads, sel, first, last, lengths, table, q,
        bd, out, ws, ws_bytes, NULL)


@pytest.mark.parametrize("sfx", ["bf16", "fp16"])
@pytest.mark.parametrize("call", [append, gather, decode, select])
def test_sizes_are_refused(lib, call, sfx):
    assert call(lib, sfx, head=0) == -1
    assert call(lib, sfx, head=257) == -2
    assert call(lib, sfx, page=0) == -1
    assert call(lib, sfx, page=65537) == -2
    assert call(lib, sfx, pages=-1) == -1
    assert call(lib, sfx, blocks=-1) == -1
    assert call(lib, sfx, blocks=(1 << 31)//16) == -2       # positions need 32 bits
    assert call(lib, sfx, batch=-1) == -1
    assert call(lib, sfx, heads=-1) == -1
    assert call(lib, sfx, batch=1 << 13, heads=1 << 12) == -2
    # nothing to do is fine, whatever the pointers
    assert call(lib, sfx, batch=0, lengths=NULL, table=NULL) == 0
    assert call(lib, sfx, heads=0, lengths=NULL, table=NULL) == 0


@pytest.mark.parametrize("call,names", [
    (append, ["lengths", "table", "k", "v", "kp", "vp"]),
    (gather, ["lengths", "table", "k", "v", "kp", "vp"]),
    (decode, ["lengths", "table", "q", "kp", "vp", "out", "ws"]),
    (select, ["lengths", "table", "q", "bd", "out", "ws"])])
def test_missing_and_unaligned_pointers_are_refused(lib, call, names):
    for name in names:
        assert call(lib, **{name: NULL}) == -1, name
        assert call(lib, **{name: ODD}) == -3, name


def test_formats_scales_and_workspaces_are_checked(lib):
    for call in (append, gather, decode):
        assert call(lib, fmt=2) == -1
        assert call(lib, fmt=-1) == -1
        assert call(lib, fmt=1) == -1                       # 8-bit pages without scales
        assert call(lib, fmt=1, ks=FAKE) == -1
    assert append(lib, new=-1) == -1
    assert append(lib, new=0, k=NULL, v=NULL) == 0
    assert append(lib, pages=0) == -1 and append(lib, blocks=0) == -1
    assert append(lib, bd=ODD) == -3 and append(lib, status=ODD) == -3
    assert gather(lib, seq=-1) == -1
    assert gather(lib, seq=0, k=NULL, v=NULL) == 0
    assert decode(lib, group=0) == 0 and decode(lib, group=-1) == -1
    assert decode(lib, sel=-1) == -1
    assert decode(lib, sel=3) == -1                         # a count without a list
    need = lib.nntile_b200_paged_decode_sdpa_workspace_bytes(64, 16, 4, 2, 2, 2, 0)
    assert need > 0
    assert decode(lib, ws_bytes=need - 1) == -4
    assert decode(lib, ws=ctypes.c_void_p((1 << 20) + 8)) == -3
    assert select(lib, sel=0, first=0, last=0, out=NULL) == 0
    assert select(lib, sel=0) == -1
    assert select(lib, sel=3, first=2, last=2) == -1
    assert select(lib, first=-1) == -1 and select(lib, last=-1) == -1
    need = lib.nntile_b200_paged_select_workspace_bytes(4, 2, 2)
    assert need > 0
    assert select(lib, ws_bytes=need - 1) == -4
    assert lib.nntile_b200_paged_decode_sdpa_workspace_bytes(0, 16, 4, 2, 2, 2, 0) == 0
    assert lib.nntile_b200_paged_decode_sdpa_workspace_bytes(64, 16, 4, 2, -2, 2, 0) == 0
    assert lib.nntile_b200_paged_select_workspace_bytes(4, -2, 2) == 0


def test_page_buffers_are_checked():
    k = torch.zeros((4, 2, 16, 64), dtype=torch.bfloat16)
    codes = torch.zeros((4, 2, 16, 64), dtype=torch.uint8)
    scales = torch.zeros((4, 2, 16), dtype=torch.uint8)
    bounds = torch.zeros((4, 2, 2, 64), dtype=torch.bfloat16)
    sdpa.KVPages(k, k, bounds=bounds)
    sdpa.KVPages(codes, codes, scales, scales, bounds)
    with pytest.raises(ValueError):
        sdpa.KVPages(k, k[:2])
    with pytest.raises(ValueError):
        sdpa.KVPages(k, k, scales, scales)
    with pytest.raises(ValueError):
        sdpa.KVPages(codes, codes, scales)
    with pytest.raises(ValueError):
        sdpa.KVPages(k, k, bounds=bounds[:, :, :1])
    with pytest.raises(ValueError):
        sdpa.KVPages(k, k, bounds=bounds.half())
    with pytest.raises(TypeError):
        sdpa.KVPages(k.float(), k.float())


def test_function_arguments_are_checked():
    k = torch.zeros((4, 2, 16, 64), dtype=torch.bfloat16)
    pages = sdpa.KVPages(k, k)
    rows = torch.zeros((2, 3, 5, 64), dtype=torch.bfloat16)
    q = torch.zeros((2, 4, 3, 1, 64), dtype=torch.bfloat16)
    lens = torch.zeros(3, dtype=torch.int32)
    table = torch.zeros((3, 2), dtype=torch.int32)
    with pytest.raises(ValueError):
        sdpa.paged_append(pages, lens, table, rows[:1], rows[:1])
    with pytest.raises(ValueError):
        sdpa.paged_append(pages, lens[:2], table, rows, rows)
    with pytest.raises(TypeError):
        sdpa.paged_append(pages, lens.long(), table, rows, rows)
    with pytest.raises(TypeError):
        sdpa.paged_append(pages, lens, table, rows.half(), rows.half())
    with pytest.raises(ValueError):
        sdpa.paged_append(pages, lens, table, rows, rows, new_lens=lens[:1])
    with pytest.raises(ValueError):
        sdpa.paged_append(pages, lens, table, rows, rows, status=lens)
    with pytest.raises(ValueError):
        sdpa.paged_gather(pages, lens, table, rows, rows[:, :, :2])
    with pytest.raises(ValueError):
        sdpa.paged_decode(q[:, :, :, :, :32], pages, lens, table)
    with pytest.raises(TypeError):
        sdpa.paged_decode(q.half(), pages, lens, table)
    with pytest.raises(ValueError):
        sdpa.paged_decode(q, pages, lens, table, selected=torch.zeros((2, 3, 0), dtype=torch.int32))
    with pytest.raises(ValueError):
        sdpa.paged_select(q, pages, lens, table, 2)         # no bounds
    # tensors that are not on a GPU
    with pytest.raises(ValueError):
        sdpa.paged_append(pages, lens, table, rows, rows)
    with pytest.raises(ValueError):
        sdpa.paged_decode(q, pages, lens, table)


def test_cache_bookkeeping_refuses_before_it_changes_anything(monkeypatch):
    """Pages are handed out on the host: a call that does not fit leaves the cache as it was."""
    calls = []
    monkeypatch.setattr(sdpa, "paged_append", lambda *a, **k: calls.append(a))
    c = sdpa.PagedKVCache(5, 16, 2, 2, 64, max_blocks=4, device="cpu")

    def rows(n, dtype=torch.bfloat16):
        return torch.zeros((2, 2, n, 64), dtype=dtype)
    c.append(rows(20), rows(20), [20, 3])
    assert c.free_pages == 2 and len(c) == 20 and c.sequence_lengths() == [20, 3]
    assert c.lengths.tolist() == [20, 3]
    assert (c.block_table >= 0).sum(1).tolist() == [2, 1]
    for bad in ([45, 0], [33, 14]):                         # table, pool
        with pytest.raises(ValueError):
            c.append(rows(45), rows(45), bad)
        assert c.free_pages == 2 and c.sequence_lengths() == [20, 3] and len(calls) == 1
    with pytest.raises(ValueError):
        c.append(rows(2), rows(2), [3, 0])
    with pytest.raises(ValueError):
        c.append(rows(2)[:, :1], rows(2)[:, :1])
    with pytest.raises(TypeError):
        c.append(rows(2, torch.float16), rows(2, torch.float16))
    assert len(calls) == 1

    def fails(*a, **k):
        raise ValueError("rows on another device")
    with monkeypatch.context() as m:                        # the call itself is refused
        m.setattr(sdpa, "paged_append", fails)
        with pytest.raises(ValueError):
            c.append(rows(30), rows(30), [10, 30])
    assert c.free_pages == 2 and c.sequence_lengths() == [20, 3] and c.lengths.tolist() == [20, 3]
    used = set(c.block_table[0, :2].tolist())
    c.release(0)
    assert c.free_pages == 4 and c.sequence_lengths() == [0, 3] and c.lengths.tolist() == [0, 3]
    c.append(rows(17), rows(17), [0, 17])
    assert c.block_table[1, :2].tolist()[1] in used         # a released page is used again
    c.clear()
    assert c.free_pages == 5 and len(c) == 0
