"""The build without what its Python extension needs, and extensions built for something else. The compiler of the kernels is
a stand-in that leaves empty files. No GPU needed."""

from __future__ import annotations

import os
import subprocess
import sys
import sysconfig

import pytest
import torch

from conftest import ROOT
from unblend_b200 import _lib, build


@pytest.fixture
def tree(tmp_path, monkeypatch):
    """A source tree of one kernel and an extension, with an older build's extension in place."""
    for name in ("csrc", "lib", "obj"):
        (tmp_path / name).mkdir()
    (tmp_path / "csrc" / "a.cu").write_text("")
    (tmp_path / "csrc" / "tensor_lists.cpp").write_text("extern \"C\" int f() { return 1; }\n")
    (tmp_path / "lib" / "tensor_lists.so").write_text("old")
    (tmp_path / "lib" / "tensor_lists.so.torch").write_text("old")
    nvcc = tmp_path / "nvcc"
    nvcc.write_text('#!/bin/sh\nwhile [ "$1" != -o ]; do shift; done\n: > "$2"\n')
    nvcc.chmod(0o755)
    monkeypatch.setenv("NVCC", str(nvcc))
    monkeypatch.delenv("CXX", raising=False)
    for name, sub in (("CSRC", "csrc"), ("LIBDIR", "lib"), ("OBJDIR", "obj")):
        monkeypatch.setattr(build, name, str(tmp_path / sub))
    return tmp_path


def _made(tree):
    """Whether library and extension are there; the library always is, with its stamp."""
    assert (tree / "lib" / "libunblend_b200.so").exists()
    assert (tree / "lib" / "libunblend_b200.digest").read_text().strip() == build.source_digest()
    so, stamp = tree / "lib" / "tensor_lists.so", tree / "lib" / "tensor_lists.so.torch"
    assert so.exists() == stamp.exists()
    return so.exists()


def test_without_a_compiler(tree, monkeypatch, capsys):
    monkeypatch.setenv("CXX", str(tree / "no-such-compiler"))
    build.build()
    assert not _made(tree) and "no-such-compiler is missing" in capsys.readouterr().err


def test_without_python_headers(tree, monkeypatch, capsys):
    get_path = sysconfig.get_path
    monkeypatch.setattr(sysconfig, "get_path", lambda n, *a, **k: str(tree) if n == "include" else get_path(n, *a, **k))
    build.build()
    assert not _made(tree) and "Python.h is missing" in capsys.readouterr().err


def test_without_torch(tree):
    code = ("import sys; sys.modules['torch'] = None\n"
            "from unblend_b200 import build\n"
            f"build.CSRC, build.LIBDIR, build.OBJDIR = (r'{tree}' + '/' + x for x in ('csrc', 'lib', 'obj'))\n"
            "print(build.build())\n")
    got = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True)
    assert got.returncode == 0, got.stderr
    assert got.stdout.strip().endswith("libunblend_b200.so") and "torch" in got.stderr
    assert not _made(tree)


def test_an_extension_that_does_not_compile(tree):
    """An error, after the library is in place, and no older extension beside it."""
    (tree / "csrc" / "tensor_lists.cpp").write_text("#error no\n")
    with pytest.raises(RuntimeError, match="failed for"):
        build.build()
    assert not _made(tree)


def test_it_is_built_again_for_another_torch(tree, monkeypatch):
    build.build()
    so = tree / "lib" / "tensor_lists.so"
    assert _made(tree) and so.read_bytes() != b"old"
    assert (tree / "lib" / "tensor_lists.so.torch").read_text() == build.extension_stamp()
    at = os.stat(so).st_mtime_ns
    build.build()
    assert os.stat(so).st_mtime_ns == at
    monkeypatch.setattr(torch, "__version__", "1.2.3")
    build.build()
    assert os.stat(so).st_mtime_ns != at and "1.2.3" in build.extension_stamp()


def test_another_build_is_not_loaded(tmp_path, monkeypatch):
    _lib.load()
    monkeypatch.setattr(_lib, "LIB_PATH", str(tmp_path / "libunblend_b200.so"))
    monkeypatch.setattr(_lib, "_tensor_lists", None)
    with pytest.raises(RuntimeError, match="not built"):
        _lib.tensor_lists()
    (tmp_path / "tensor_lists.so").write_text("no library")
    (tmp_path / "tensor_lists.so.torch").write_text("torch 1.2.3, cpython-27")
    with pytest.raises(RuntimeError, match="was built for torch 1.2.3, cpython-27"):
        _lib.tensor_lists()
