"""What the build makes, and when: the C library without torch; the binding of
the paged operators again whenever torch, the interpreter or the command that it
was compiled with change. Compilers are stood in for."""

from __future__ import annotations

import subprocess
import sys
import types

import pytest
import torch

from dequant_project_b200 import build as B
from dequant_project_b200 import paged_ops


@pytest.fixture
def tree(tmp_path, monkeypatch):
    """An empty tree with one source; every command writes its output file."""
    (tmp_path / "csrc").mkdir()
    (tmp_path / "csrc" / "a.cu").write_text("")
    (tmp_path / "binding.cpp").write_text("")
    runs = []

    def run(cmd, **kw):
        runs.append(cmd)
        out = cmd[cmd.index("-o") + 1]
        open(out, "w").close()
        return types.SimpleNamespace(returncode=0, stdout="", stderr="")

    monkeypatch.setattr(subprocess, "run", run)
    monkeypatch.setattr(B, "nvcc", lambda: "/usr/local/cuda/bin/nvcc")
    for name, path in (("CSRC", "csrc"), ("OUT", "lib.so"), ("OBJ_DIR", "_build"), ("BINDING", "binding.cpp"),
                       ("BINDING_OUT", "_paged_binding.so"), ("INCLUDE", "include")):
        monkeypatch.setattr(B, name, tmp_path / path)
    return types.SimpleNamespace(path=tmp_path, runs=runs)


def test_the_library_is_built_without_torch(tree, monkeypatch, capsys):
    monkeypatch.setitem(sys.modules, "torch", None)  # import torch raises
    assert B.build() == tree.path / "lib.so"
    assert (tree.path / "lib.so").exists() and not (tree.path / "_paged_binding.so").exists()
    assert "binding is not built: torch cannot be imported" in capsys.readouterr().err


@pytest.mark.parametrize("missing", ["compiler", "headers"])
def test_the_library_is_built_without_a_cpp_toolchain(tree, monkeypatch, capsys, missing):
    if missing == "compiler":
        monkeypatch.setenv("CXX", "no-such-compiler")
    else:
        monkeypatch.setattr(B.sysconfig, "get_paths", lambda: {"include": str(tree.path / "nowhere")})
    assert B.build() == tree.path / "lib.so"
    assert (tree.path / "lib.so").exists() and not (tree.path / "_paged_binding.so").exists()
    assert "binding is not built" in capsys.readouterr().err


def test_a_binding_that_fails_to_compile_leaves_the_library(tree, monkeypatch):
    run = subprocess.run

    def fail(cmd, **kw):
        r = run(cmd, **kw)
        if str(tree.path / "binding.cpp") in cmd:
            r.returncode, r.stderr = 1, "no such type"
        return r

    monkeypatch.setattr(subprocess, "run", fail)
    with pytest.raises(RuntimeError, match="no such type"):
        B.build()
    assert (tree.path / "lib.so").exists() and not (tree.path / "_paged_binding.so").exists()


def test_the_binding_follows_what_it_was_built_with(tree, monkeypatch):
    def compiled():
        n = len(tree.runs)
        B.build_binding()
        return len(tree.runs) > n

    assert compiled() and not compiled()
    monkeypatch.setattr(torch, "__version__", "99.0")
    assert compiled() and not compiled()
    monkeypatch.setattr(B.sysconfig, "get_config_var", lambda name: "cpython-399")
    assert compiled() and not compiled()
    monkeypatch.setenv("CXX", "gcc")
    assert compiled() and not compiled()


def test_another_torch_is_refused(monkeypatch):
    monkeypatch.setattr(paged_ops, "_bound", None)
    monkeypatch.setattr(torch, "__version__", "99.0")
    with pytest.raises(ImportError, match="built for torch .*, this is 99.0"):
        paged_ops._binding()


def test_the_reason_of_a_failed_import_is_told(monkeypatch):
    import dequant_project_b200
    monkeypatch.setattr(paged_ops, "_bound", None)
    monkeypatch.delattr(dequant_project_b200, "_paged_binding", raising=False)
    monkeypatch.setitem(sys.modules, "dequant_project_b200._paged_binding", None)
    with pytest.raises(ImportError, match="halted"):
        paged_ops._binding()
