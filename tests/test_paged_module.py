"""The extension module of the paged calls: when it is built again, and what is said when it does
not load."""
import sys
import warnings

import pytest

import nntile_b200
from nntile_b200 import build, sdpa


def test_another_torch_or_python_builds_the_module_again(tmp_path, monkeypatch):
    build.build()
    assert not build._torch_module_stale()
    with monkeypatch.context() as m:
        m.setattr(build, "_torch_version", lambda: "Python 3.0 torch 1.0")
        assert build._torch_module_stale()
    with monkeypatch.context() as m:
        m.setattr(build, "TORCH_STAMP", str(tmp_path / "none"))
        assert build._torch_module_stale()
    assert not build._torch_module_stale()


def test_a_module_that_does_not_load_is_said(tmp_path, monkeypatch):
    monkeypatch.setitem(sys.modules, "nntile_b200._paged_torch", None)
    monkeypatch.delattr(nntile_b200, "_paged_torch", raising=False)
    there = tmp_path / "_paged_torch.so"
    there.write_bytes(b"")
    monkeypatch.setattr(build, "TORCH_MODULE", str(there))
    with pytest.warns(RuntimeWarning, match="does not load"):
        assert sdpa._load_paged_torch() is None
    there.unlink()                           # never built: everything goes through ops
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        assert sdpa._load_paged_torch() is None
