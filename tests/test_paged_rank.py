"""The search for the last selected block's score ends on any scores: host check of the
arithmetic that the ranking kernel does it with."""
import os
import shutil
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))


def test_the_search_for_a_rank_ends(tmp_path):
    if shutil.which("g++") is None:
        pytest.skip("no g++")
    exe = str(tmp_path / "paged_rank_check")
    subprocess.run(["g++", "-std=c++17", "-Wall", "-o", exe,
                    os.path.join(HERE, "paged_rank_check.cc")], check=True)
    assert subprocess.run([exe], timeout=60).returncode == 0
