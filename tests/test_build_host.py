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


@needs_nvcc
def test_the_binding_is_built_again_for_another_torch(tree, monkeypatch):
    """Its name says nothing of what it was compiled against: a key beside it does.
    The same key leaves it as it is; an upgrade of torch, Python or the compiler,
    or a key that is not there, does not."""
    torch = tree / "torch"
    (torch / "include" / "torch").mkdir(parents=True)
    (torch / "include" / "torch" / "version.h").write_text('#define TORCH_VERSION "x"\n')
    for lib in ("torch_python", "torch_cpu", "c10"):
        (torch / "lib").mkdir(exist_ok=True)
        subprocess.run(["g++", "-shared", "-x", "c++", "/dev/null", "-o", str(torch / "lib" / f"lib{lib}.so")], check=True)
    spec = importlib.util.spec_from_file_location("torch", torch / "__init__.py", submodule_search_locations=[str(torch)])
    find = importlib.util.find_spec
    monkeypatch.setattr(importlib.util, "find_spec", lambda name, *a: spec if name == "torch" else find(name, *a))
    made, (src, so) = [], (tree / "src" / "binding.cpp", tree / "_binding.so")
    src.write_text(src.read_text() + 'extern "C" const char *release() { return REMORA_TORCH_RELEASE; }\n')

    def build(version):
        (torch / "version.py").write_text(f"__version__ = '{version}'\n")
        b.build()
        made.append(so.stat().st_mtime_ns)
        assert version.encode() in so.read_bytes()

    for version in ("1.0", "1.0", "2.0+x"):
        build(version)
    assert made[0] == made[1] < made[2]
    monkeypatch.setattr(b.sysconfig, "get_config_var", lambda name: "another-python")
    build("2.0+x")
    assert made[2] < made[3]
    (tree / "build" / "binding.key").unlink()
    build("2.0+x")
    assert made[3] < made[4]


def test_a_binding_for_another_torch_is_refused(monkeypatch):
    from remora_b200 import _binding, ops
    from remora_b200.errors import RemoraB200Error

    assert ops._binding() is _binding
    monkeypatch.setattr(ops, "_binding_module", None)
    monkeypatch.setattr(_binding, "torch_release", "0.1")
    with pytest.raises(RemoraB200Error, match="built for torch 0.1.*csrc.build"):
        ops._binding()
