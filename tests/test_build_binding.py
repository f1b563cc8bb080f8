"""The build of the operators' torch binding (mast3r_runtime_b200/build.py): when it is left out and
when it is made anew.  The compiler is replaced; torch is a folder made here."""

from __future__ import annotations

import os
from types import SimpleNamespace

import pytest

from mast3r_runtime_b200 import build as b


@pytest.fixture
def tree(tmp_path, monkeypatch):
    """A torch with CUDA libraries and headers, an older binding source, an empty package folder."""
    root = tmp_path / "torch"
    for name in ("lib/libtorch_cuda.so", "lib/libc10_cuda.so", "lib/libtorch_python.so", "include/ATen/ATen.h",
                 "include/torch/csrc/Dtype.h", "__init__.py"):
        (root / name).parent.mkdir(parents=True, exist_ok=True)
        (root / name).write_text("")
    (root / "version.py").write_text("__version__ = '1'\n")
    python = tmp_path / "python"
    python.mkdir()
    (python / "Python.h").write_text("")
    build_dir = tmp_path / "pkg" / "_build"
    build_dir.mkdir(parents=True)
    source = tmp_path / "torch_ops.cpp"
    source.write_text("")
    os.utime(source, (1, 1))
    for name, value in (("BUILD", build_dir), ("TORCH_LIB", tmp_path / "pkg" / "_torch_ops.so"), ("BINDING", source),
                        ("TORCH_STAMP", tmp_path / "pkg" / "_torch_ops.stamp")):
        monkeypatch.setattr(b, name, value)
    made = []

    def run(cmd, **kw):
        made.append(cmd)
        with open(cmd[cmd.index("-o") + 1], "w") as f:
            f.write(f"build {len(made)}")
        return SimpleNamespace(returncode=0, stdout="", stderr="")

    monkeypatch.setattr(b.subprocess, "run", run)
    monkeypatch.setattr(b.importlib.util, "find_spec", lambda name: SimpleNamespace(origin=str(root / "__init__.py")))
    paths = dict(b.sysconfig.get_paths(), include=str(python))
    monkeypatch.setattr(b.sysconfig, "get_paths", lambda: paths)
    return SimpleNamespace(root=root, python=python, made=made, monkeypatch=monkeypatch)


def test_built_once_and_kept(tree):
    assert b.build_torch_ops() == b.TORCH_LIB and len(tree.made) == 1
    assert b.build_torch_ops() == b.TORCH_LIB and len(tree.made) == 1


def test_another_torch_or_python_builds_anew(tree):
    b.build_torch_ops()
    (tree.root / "version.py").write_text("__version__ = '2'\n")
    b.build_torch_ops()
    assert len(tree.made) == 2
    tree.monkeypatch.setattr(b.sysconfig, "get_config_var", lambda name: "cpython-399")
    b.build_torch_ops()
    b.build_torch_ops()
    assert len(tree.made) == 3


def test_a_binding_without_a_stamp_is_built_anew(tree):
    b.TORCH_LIB.write_text("made for some torch")
    os.utime(b.TORCH_LIB)
    b.build_torch_ops()
    assert len(tree.made) == 1 and b.TORCH_LIB.read_text() == "build 1"
    # the stamp travels with the binding, not with the objects
    assert b.TORCH_STAMP.exists() and b.TORCH_STAMP.parent == b.TORCH_LIB.parent


@pytest.mark.parametrize("missing", ["lib/libtorch_cuda.so", "lib/libc10_cuda.so", "include/ATen/ATen.h", "Python.h",
                                     "torch"])
def test_left_out_where_it_cannot_be_built(tree, missing, capsys):
    """A torch without CUDA or without headers, or none: the library alone is built, and says so."""
    b.build_torch_ops()
    if missing == "torch":
        tree.monkeypatch.setattr(b.importlib.util, "find_spec", lambda name: None)
    else:
        (tree.python if missing == "Python.h" else tree.root).joinpath(missing).unlink()
    assert b.build_torch_ops() is None and len(tree.made) == 1
    assert "mast3r_runtime_b200.ops is not built" in capsys.readouterr().err
    assert not b.TORCH_LIB.exists()  # nor is one kept that does not belong to this torch
