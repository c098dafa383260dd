"""CPU: the library is built without torch, and a binding that is missing or does not load raises the package's error."""
import os
import shutil
import subprocess
import sys

import pytest

PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "xtier-go_b200")


def plan(tmp_path, python):
    """The commands of `make` in a fresh copy of the sources."""
    root = tmp_path / "repo"
    if not root.exists():
        shutil.copytree(os.path.join(PKG, "csrc"), root / "pkg" / "csrc")
        shutil.copy(os.path.join(PKG, "Makefile"), root / "pkg")
        shutil.copytree(os.path.join(PKG, "..", "include"), root / "include")
    r = subprocess.run(["make", "-n", "-C", str(root / "pkg"), f"PYTHON={python}"], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    return r.stdout


def test_make_builds_the_library_alone_without_torch(tmp_path):
    without = tmp_path / "python_without_torch"
    without.write_text(f"#!/bin/sh\nexec {sys.executable} -S -I \"$@\"\n")   # no site-packages
    without.chmod(0o755)
    out = plan(tmp_path, without)
    assert "libxtg_cuda.so" in out and "kv4_torch.cpp" not in out and "is not built" in out
    out = plan(tmp_path, "/nonexistent/python")
    assert "libxtg_cuda.so" in out and "kv4_torch.cpp" not in out


def test_make_builds_the_binding_with_torch(tmp_path):
    out = plan(tmp_path, sys.executable)
    assert "libxtg_cuda.so" in out and "kv4_torch.cpp" in out


def test_a_binding_that_does_not_load(xtg, monkeypatch, tmp_path):
    monkeypatch.setattr(xtg, "HERE", str(tmp_path))
    monkeypatch.setattr(xtg, "_kv4_module", None)
    with pytest.raises(xtg.XtgError, match="is missing"):
        xtg.kv4_load(*[None] * 5)
    (tmp_path / "_kv4_torch.so").write_bytes(b"not a library")
    with pytest.raises(xtg.XtgError, match="does not load"):
        xtg.kv4_load(*[None] * 5)
