"""The build's order: the library does not wait for the host module's headers.  Compilers are stood in for."""
from pathlib import Path
from types import SimpleNamespace

import pytest

from sparsefold_amd import _build


@pytest.fixture
def tree(tmp_path, monkeypatch):
  """A package to build into, and the commands that ran."""
  commands = []

  def run(cmd, **_):
    commands.append(cmd)
    failed = any(str(c).endswith("front.cpp") for c in cmd) and tree.front_fails
    if not failed:
      Path(cmd[cmd.index("-o") + 1]).write_text("built")
    return SimpleNamespace(returncode=int(failed), stderr="no such file: Python.h" if failed else "")

  tree = SimpleNamespace(commands=commands, front_fails=False, lib=tmp_path / "libsparsefold_hip.so", front=tmp_path / "_front-x.so")
  monkeypatch.setattr(_build.subprocess, "run", run)
  monkeypatch.setattr(_build, "BUILD", tmp_path / "objects")
  monkeypatch.setattr(_build, "LIB", tree.lib)
  monkeypatch.setattr(_build, "front_path", lambda: tree.front)
  return tree


def test_library_and_host_module(tree):
  assert _build.build() == tree.lib and tree.lib.exists() and tree.front.exists()
  assert len(tree.commands) == len(list(_build.CSRC.glob("*.hip"))) + 2


def test_library_without_the_headers_of_the_host_module(tree, monkeypatch, tmp_path, capsys):
  """No Python headers: the library is linked, no host module is built, and one of an earlier build does not stay."""
  tree.front.write_text("old")
  monkeypatch.setattr(_build.sysconfig, "get_paths", lambda: {"include": str(tmp_path / "none")})
  assert _build.build(verbose=True) == tree.lib and tree.lib.exists() and not tree.front.exists()
  assert not any("front.cpp" in str(c) for cmd in tree.commands for c in cmd)
  assert "no host module" in capsys.readouterr().out


def test_library_without_torch(tree, monkeypatch):
  import sys
  monkeypatch.setitem(sys.modules, "torch", None)
  assert _build.build() == tree.lib and tree.lib.exists() and not tree.front.exists()


def test_host_module_that_does_not_compile(tree):
  """An error, behind the library's link."""
  tree.front_fails = True
  with pytest.raises(RuntimeError, match="front.cpp"):
    _build.build()
  assert tree.lib.exists() and not tree.front.exists()


def test_host_modules_of_two_pythons_stand_side_by_side(monkeypatch):
  """One torch version, two interpreters, one tree: each looks for a module of its own."""
  from sparsefold_amd import _lib
  here = _lib.front_path()
  assert any(str(here).endswith(s) and s != ".so" for s in _lib.importlib.machinery.EXTENSION_SUFFIXES)
  monkeypatch.setattr(_lib.sysconfig, "get_config_var", lambda name: ".cpython-399-x86_64-linux-gnu.so")
  assert _lib.front_path() != here and _lib.front_path().parent == here.parent
