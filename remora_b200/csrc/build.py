"""Build libremora_b200.so in-tree with nvcc for sm_100a, and the Python
binding's host code (_binding.so) with the host compiler.

Usage: python -m remora_b200.csrc.build  (or build() from Python).  Object
files go to remora_b200/csrc/_build/; the shared library lands next to the
package so a plain snapshot of the repository carries it.
"""

from __future__ import annotations

import importlib.util
import os
import re
import shutil
import subprocess
import sys
import sysconfig
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

HERE = Path(__file__).resolve().parent
PKG = HERE.parent
ROOT = PKG.parent
OUT = PKG / "libremora_b200.so"
BINDING = PKG / "_binding.so"
BUILD = HERE / "_build"

SOURCES = sorted(HERE.glob("*.cu"))

CUDA_HOME = Path(os.environ.get("CUDA_HOME", "/usr/local/cuda"))
NVCC = str(CUDA_HOME / "bin" / "nvcc")
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
FLAGS = [
    "-O3",
    "-std=c++17",
    "-lineinfo",
    "-Xcompiler",
    "-fPIC",
    f"-I{ROOT / 'include'}",
    "--expt-relaxed-constexpr",
]


def _host_compiler() -> list[str]:
    # nvcc needs a host g++; prefer the system one over a CC/CXX from the
    # environment that may lack pieces of its runtime.
    for cand in ("/usr/bin/g++", shutil.which("g++")):
        if cand and Path(cand).exists():
            return ["-ccbin", cand]
    return []


def _needs_rebuild(obj: Path, src: Path) -> bool:
    if not obj.exists():
        return True
    deps = [src, *HERE.glob("*.cuh"), *(ROOT / "include").glob("*.h")]
    return any(d.stat().st_mtime > obj.stat().st_mtime for d in deps if d.exists())


def _compile(src: Path, verbose: bool) -> Path:
    obj = BUILD / (src.stem + ".o")
    if _needs_rebuild(obj, src):
        cmd = [NVCC, *_host_compiler(), *ARCH, *FLAGS, "-c", str(src), "-o", str(obj)]
        if verbose:
            print(" ".join(cmd), flush=True)
        subprocess.run(cmd, check=True)
    return obj


def _build_binding(verbose: bool) -> None:
    """_binding.so: binding.cpp against the headers of the installed torch.
    Without torch there is nothing that it could bind, and C programs need the
    library alone."""
    src = HERE / "binding.cpp"
    spec = importlib.util.find_spec("torch")
    if spec is None or not spec.submodule_search_locations:
        print("remora_b200._binding is left out: torch is not installed", file=sys.stderr, flush=True)
        return
    torch_dir = Path(next(iter(spec.submodule_search_locations)))
    cxx = _host_compiler()[1:] or ["g++"]
    # what it is compiled against: with another torch, Python or compiler its layouts differ
    release = re.search(r"__version__ = '([^']*)'", (torch_dir / "version.py").read_text())
    version = release.group(1) if release else "unknown"
    compiler = subprocess.run([*cxx, "--version"], capture_output=True, text=True, check=True).stdout.splitlines()[0]
    key = "\n".join([version, str(torch_dir), sysconfig.get_config_var("SOABI") or sys.version, " ".join(cxx), compiler])
    stamp = BUILD / "binding.key"
    if (BINDING.exists() and BINDING.stat().st_mtime >= src.stat().st_mtime
            and stamp.exists() and stamp.read_text() == key):
        return
    made = BUILD / BINDING.name
    cmd = [
        *cxx,
        "-O2",
        "-std=c++17",
        "-fPIC",
        "-shared",
        f"-I{torch_dir / 'include'}",
        f"-I{torch_dir / 'include' / 'torch' / 'csrc' / 'api' / 'include'}",
        f"-I{sysconfig.get_paths()['include']}",
        f'-DREMORA_TORCH_RELEASE="{version}"',
        str(src),
        "-o",
        str(made),
        f"-L{torch_dir / 'lib'}",
        "-ltorch_python",
        "-ltorch_cpu",
        "-lc10",
        f"-Wl,-rpath,{torch_dir / 'lib'}",
    ]
    if verbose:
        print(" ".join(cmd), flush=True)
    subprocess.run(cmd, check=True)
    # put in place as a whole, and named by its key only then
    stamp.unlink(missing_ok=True)
    os.replace(made, BINDING)
    stamp.write_text(key)


def build(verbose: bool = False, jobs: int | None = None) -> Path:
    BUILD.mkdir(exist_ok=True)
    with ThreadPoolExecutor(max_workers=jobs or min(8, os.cpu_count() or 1)) as ex:
        binding = ex.submit(_build_binding, verbose)
        objs = list(ex.map(lambda s: _compile(s, verbose), SOURCES))
    if not OUT.exists() or any(o.stat().st_mtime > OUT.stat().st_mtime for o in objs):
        cmd = [
            NVCC,
            *_host_compiler(),
            *ARCH,
            "-shared",
            "-o",
            str(OUT),
            *map(str, objs),
            f"-L{CUDA_HOME / 'lib64'}",
            "-lnvrtc",
            f"-Xlinker=-rpath,{CUDA_HOME / 'lib64'}",
        ]
        if verbose:
            print(" ".join(cmd), flush=True)
        subprocess.run(cmd, check=True)
    binding.result()  # a failure of its own, behind the library
    return OUT


if __name__ == "__main__":
    print(build(verbose="-v" in sys.argv))
