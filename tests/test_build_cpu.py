"""What the in-tree build makes of a machine without torch, its headers or a C++ compiler: host code, nothing is compiled here."""
import importlib.util
import os

import pytest

from imagecaptioner_amd import build


@pytest.fixture
def recorded(monkeypatch, tmp_path):
    """The build with its two compilations replaced by their outputs' appearance in a folder of their own."""
    ran = []

    def touch(path, what):
        with open(path, "w") as f:
            f.write("torch module for %s\0" % build._torch_name() if what == "torch module" else "")
            ran.append(what)
    monkeypatch.setattr(build, "LIB", str(tmp_path / "lib.so"))
    monkeypatch.setattr(build, "TORCH_LIB", str(tmp_path / "torch.so"))
    monkeypatch.setattr(build, "_build", lambda lib, *a, **k: touch(lib, "library"))
    monkeypatch.setattr(build, "_build_torch_module", lambda verbose: touch(build.TORCH_LIB, "torch module"))
    return ran


def test_both_parts_and_only_what_is_stale(recorded):
    assert build._torch_module_missing() is None
    assert build.build() == build.LIB and sorted(recorded) == ["library", "torch module"]
    recorded.clear()
    build.build()
    assert recorded == []
    os.utime(build.TORCH_LIB, (1, 1))
    build.build()
    assert recorded == ["torch module"]
    recorded.clear()
    os.utime(build.LIB, (1, 1))
    build.build()
    assert recorded == ["library"]
    recorded.clear()
    build.build(force=True)
    assert sorted(recorded) == ["library", "torch module"]


@pytest.mark.parametrize("what", ["torch", "headers", "compiler"])
def test_the_library_is_built_without_torch(recorded, monkeypatch, tmp_path, capsys, what):
    if what == "torch":
        monkeypatch.setattr(importlib.util, "find_spec", lambda name: None)
    elif what == "headers":
        spec = importlib.util.spec_from_file_location("torch", str(tmp_path / "__init__.py"))
        monkeypatch.setattr(importlib.util, "find_spec", lambda name: spec)
    else:
        monkeypatch.setattr(build, "CXX", str(tmp_path / "none"))
    assert build.build(force=True) == build.LIB and recorded == ["library"]
    assert "without the torch module" in capsys.readouterr().out
    build.build()                                                # and it is not stale for the module's absence
    assert recorded == ["library"]


def test_another_torch(recorded, monkeypatch):
    """A module that was built against another torch is stale, and refused where it is loaded all the same."""
    import torch

    from imagecaptioner_amd import TagPipeError, replies
    assert build._torch_name() == "%s %s" % (torch.__version__, torch.version.git_version)
    build.build()
    recorded.clear()
    assert not build._torch_module_stale()
    monkeypatch.setattr(build, "_torch_name", lambda: "9.9.9 abc")
    assert build._torch_module_stale() and not build._stale()
    build.build()
    assert recorded == ["torch module"] and not build._torch_module_stale()
    monkeypatch.setattr(replies, "_native_module", None)
    assert replies._native().built_for.endswith(torch.version.git_version)
    monkeypatch.setattr(replies, "_native_module", None)
    monkeypatch.setattr(torch.version, "git_version", "abc")
    with pytest.raises(TagPipeError, match="abc, and the module is a torch module for"):
        replies._native()
