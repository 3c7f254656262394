"""What the incremental build compiles again: everything whose source, headers or compiler flags (which stand in build.py) are newer."""
import importlib.util
import os
import shutil

import pytest

import adcdiff

PACKAGE = os.path.dirname(os.path.abspath(adcdiff._lib.__file__))


@pytest.fixture
def tree(tmp_path, monkeypatch):
    """a copy of the sources with an up-to-date build, whose compilers only write down what they are asked for"""
    pkg = tmp_path / "pkg"
    shutil.copytree(os.path.join(PACKAGE, "csrc"), pkg / "csrc")
    shutil.copytree(os.path.join(os.path.dirname(PACKAGE), "include"), tmp_path / "include")
    shutil.copy(os.path.join(PACKAGE, "build.py"), pkg / "build.py")
    spec = importlib.util.spec_from_file_location("build_under_test", str(pkg / "build.py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    made = []

    def run(cmd, check=True):
        out = cmd[cmd.index("-o") + 1] if "-o" in cmd else cmd[-1]
        made.append(os.path.basename(out))
        open(out, "a").close()
        os.utime(out)
    monkeypatch.setattr(mod.subprocess, "run", run)
    monkeypatch.setattr(mod.shutil, "which", lambda name: "/bin/" + name)
    old = os.path.getmtime(PACKAGE) - 10000
    for base, _, files in os.walk(str(tmp_path)):
        for f in files:
            os.utime(os.path.join(base, f), (old, old))
    mod.build_library()
    everything = sorted(made)
    made.clear()
    return mod, pkg, made, everything


def _touch(path):
    os.utime(str(path))
    later = os.path.getmtime(str(path)) + 5
    os.utime(str(path), (later, later))


def test_nothing_changed(tree):
    mod, _, made, everything = tree
    assert {s.replace(".hip", ".o") for s, _ in mod.SOURCES} | {"libadcdiff.so", "libadcdiff_torch.so"} <= set(everything)
    mod.build_library()
    assert made == []


def test_one_source(tree):
    mod, pkg, made, _ = tree
    _touch(pkg / "csrc" / "grad_norm.hip")
    mod.build_library()
    assert made == ["grad_norm.o", "libadcdiff.so"]


@pytest.mark.parametrize("changed", ["build.py", "csrc/row_access.h"])
def test_flags_and_headers(tree, changed):
    mod, pkg, made, _ = tree
    _touch(pkg / changed)
    mod.build_library()
    assert {s.replace(".hip", ".o") for s, _ in mod.SOURCES} | {"libadcdiff.so"} <= set(made)
    assert ("libadcdiff_torch.so" in made) == (changed == "build.py")


def test_forced(tree):
    mod, _, made, everything = tree
    mod.build_library(force=True)
    assert set(everything) <= set(made)


def test_entry_point_compiles_every_time(monkeypatch):
    """__graft_entry__.build() answers whether the sources compile, so a library that is already there does not count"""
    import __graft_entry__ as entry
    asked = []

    class Module:
        @staticmethod
        def build_library(force=False, verbose=False):
            asked.append(force)
            return "library"
    monkeypatch.setattr(importlib.util, "module_from_spec", lambda spec: Module)
    monkeypatch.setattr(importlib.util, "spec_from_file_location", lambda *a: type("S", (), {"loader": type("L", (), {"exec_module": staticmethod(lambda m: None)})}))
    entry.build()
    assert asked == [True]
