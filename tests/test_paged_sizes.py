"""Paged calls at the largest sizes they take, as far as that needs no GPU: the arithmetic of the
kernels on the host, and refusals."""
import os
import shutil
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))


def test_splits_of_a_list_take_all_of_it(tmp_path):
    if shutil.which("g++") is None:
        pytest.skip("no g++")
    exe = str(tmp_path / "paged_split_check")
    subprocess.run(["g++", "-std=c++17", "-Wall", "-o", exe,
                    os.path.join(HERE, "paged_split_check.cc")], check=True)
    assert subprocess.run([exe], timeout=60).returncode == 0
