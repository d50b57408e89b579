"""build.py's order of things, with stand-ins for the compilers that only write their output files."""
import builtins
import importlib.util
import os
import stat

import pytest

from conftest import PKG, ROOT

TOOL = """#!/bin/sh
while [ $# -gt 0 ]; do
  if [ "$1" = "-o" ]; then echo made > "$2"; fi
  shift
done
exit %d
"""


def _tool(path, code):
    path.write_text(TOOL % code)
    path.chmod(path.stat().st_mode | stat.S_IXUSR)
    return str(path)


@pytest.fixture
def build(tmp_path, monkeypatch):
    spec = importlib.util.spec_from_file_location("build_under_test", os.path.join(ROOT, PKG, "build.py"))
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    monkeypatch.setattr(module, "HERE", str(tmp_path))
    monkeypatch.setattr(module, "LIB", str(tmp_path / "lib.so"))
    monkeypatch.setattr(module, "BIND_LIB", str(tmp_path / "bind.so"))
    monkeypatch.setattr(module, "HIPCC", _tool(tmp_path / "hipcc", 0))
    monkeypatch.setenv("CXX", _tool(tmp_path / "cxx", 0))
    module.where = tmp_path
    return module


def test_library_and_binding(build):
    assert build.build() == build.LIB
    assert os.path.exists(build.LIB) and os.path.exists(build.BIND_LIB)


def test_the_library_needs_no_torch(build, monkeypatch):
    real = builtins.__import__

    def without_torch(name, *args, **kw):
        if name == "torch":
            raise ModuleNotFoundError("No module named 'torch'", name="torch")
        return real(name, *args, **kw)

    monkeypatch.setattr(builtins, "__import__", without_torch)
    assert build.build() == build.LIB
    assert os.path.exists(build.LIB) and not os.path.exists(build.BIND_LIB)


@pytest.mark.parametrize("cxx", ["fails", "missing"])
def test_a_failed_binding_is_raised_with_the_library_in_place(build, monkeypatch, cxx):
    monkeypatch.setenv("CXX", _tool(build.where / "bad", 1) if cxx == "fails" else str(build.where / "none"))
    with pytest.raises(RuntimeError, match="binding"):
        build.build()
    assert os.path.exists(build.LIB) and not os.path.exists(build.BIND_LIB)


def test_a_failed_library_is_raised(build, monkeypatch):
    monkeypatch.setattr(build, "HIPCC", _tool(build.where / "bad", 1))
    with pytest.raises(RuntimeError, match="hipcc failed"):
        build.build()
    assert not os.path.exists(build.LIB)
