"""The in-tree build, on small sources of its own: what it makes without torch."""

from __future__ import annotations

import ctypes
import importlib.util
import shutil
import subprocess

import pytest

from remora_b200.csrc import build as b

needs_nvcc = pytest.mark.skipif(shutil.which(str(b.NVCC)) is None, reason="nvcc is not installed")


@pytest.fixture
def tree(tmp_path, monkeypatch):
    """The build's paths in a tree with one source and no binding."""
    (tmp_path / "src").mkdir()
    (tmp_path / "src" / "one.cu").write_text('extern "C" int answer() { return 42; }\n')
    (tmp_path / "src" / "binding.cpp").write_text("#include <torch/version.h>\nconst char *torch_is = TORCH_VERSION;\n")
    for name, path in dict(HERE=tmp_path / "src", OUT=tmp_path / "lib.so", BINDING=tmp_path / "_binding.so",
                           BUILD=tmp_path / "build").items():
        monkeypatch.setattr(b, name, path)
    monkeypatch.setattr(b, "SOURCES", [tmp_path / "src" / "one.cu"])
    return tmp_path


@needs_nvcc
def test_the_library_is_built_without_torch(tree, monkeypatch, capfd):
    find = importlib.util.find_spec
    monkeypatch.setattr(importlib.util, "find_spec", lambda name, *a: None if name == "torch" else find(name, *a))
    assert b.build() == tree / "lib.so"
    assert ctypes.CDLL(str(tree / "lib.so")).answer() == 42
    assert not (tree / "_binding.so").exists() and "torch is not installed" in capfd.readouterr().err


@needs_nvcc
def test_a_binding_that_does_not_compile_is_an_error_behind_the_library(tree):
    (tree / "src" / "binding.cpp").write_text("#error no\n")
    with pytest.raises(subprocess.CalledProcessError):
        b.build()
    assert (tree / "lib.so").exists()
