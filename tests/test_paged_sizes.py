"""Paged calls at the largest sizes they take, as far as that needs no GPU: the arithmetic of the
kernels on the host, and refusals."""
import ctypes
import os
import shutil
import subprocess

import pytest

from nntile_b200 import _lib, build

HERE = os.path.dirname(os.path.abspath(__file__))


def test_splits_of_a_list_take_all_of_it(tmp_path):
    if shutil.which("g++") is None:
        pytest.skip("no g++")
    exe = str(tmp_path / "paged_split_check")
    subprocess.run(["g++", "-std=c++17", "-Wall", "-o", exe,
                    os.path.join(HERE, "paged_split_check.cc")], check=True)
    assert subprocess.run([exe], timeout=60).returncode == 0


@pytest.mark.parametrize("sfx", ["bf16", "fp16"])
def test_selections_of_more_blocks_than_the_loops_count_are_refused(sfx):
    if not os.path.exists(_lib.LIB_PATH):
        build.build()
    lib = _lib.load()
    fake = ctypes.c_void_p(1 << 20)          # never dereferenced: the calls are refused
    fn = getattr(lib, f"nntile_b200_paged_select_{sfx}")

    def select(blocks, selected):
        return fn(None, 64, 1, 8, blocks, 1, 1, 1, selected, 0, 0, fake, fake, fake, fake, fake,
                  fake, 1 << 62, None)
    for big in ((1 << 30) + 1, (1 << 31) - 20000, (1 << 31) - 1):
        assert select(big, 4) == -2
        assert select(4, big) == -2
        assert lib.nntile_b200_paged_select_workspace_bytes(big, 1, 1) == 0
    assert lib.nntile_b200_paged_select_workspace_bytes(1 << 30, 1, 1) > 0
