"""The extension module of the paged calls: when it is built again."""
from nntile_b200 import build


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
