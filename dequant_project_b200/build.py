"""Build libdequant_b200.so in-tree (sm_100a only).

    python -m dequant_project_b200.build [--force] [--verbose-ptxas]

Each ``csrc/*.cu`` is compiled by nvcc for ``arch=compute_100a,code=sm_100a``
with ``-lineinfo`` and linked into ``dequant_project_b200/libdequant_b200.so``
next to this file (static CUDA runtime, no torch dependency). The shared
library is the product's C ABI (include/dequant_b200.h); the Python package
loads it with ctypes. The paged-cache operators' calls are also bound natively
(``binding/paged_binding.cpp``, built against the installed torch into
``_paged_binding.so``).
"""

from __future__ import annotations

import concurrent.futures as cf
import os
import shutil
import subprocess
import sys
from pathlib import Path

PKG = Path(__file__).resolve().parent
CSRC = PKG / "csrc"
INCLUDE = PKG.parent / "include"
OUT = PKG / "libdequant_b200.so"
OBJ_DIR = PKG / "_build"
BINDING = PKG / "binding" / "paged_binding.cpp"
BINDING_OUT = PKG / "_paged_binding.so"
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]


def nvcc() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and Path(cand).exists():
            return cand
    raise RuntimeError("nvcc not found: set NVCC or put CUDA's bin directory on PATH")


def sources():
    return sorted(CSRC.glob("*.cu"))


def _stale(paths) -> bool:
    if not OUT.exists():
        return True
    t = OUT.stat().st_mtime
    deps = list(paths) + list(CSRC.glob("*.cuh")) + list(CSRC.glob("*.h")) + list(INCLUDE.glob("*.h"))
    return any(p.stat().st_mtime > t for p in deps)


def _compile(src: Path, verbose_ptxas: bool) -> Path:
    obj = OBJ_DIR / (src.stem + ".o")
    cmd = [nvcc(), *ARCH, "-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC",
           "-I", str(CSRC), "-I", str(INCLUDE), "-c", str(src), "-o", str(obj)]
    if verbose_ptxas:
        cmd += ["-Xptxas", "-v"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"nvcc failed for {src.name}:\n{r.stdout}\n{r.stderr}")
    if verbose_ptxas:
        sys.stderr.write(r.stderr)
    return obj


def build_binding(force: bool = False) -> Path:
    """The native binding of the paged operators (g++, torch's headers)."""
    deps = [BINDING, *INCLUDE.glob("*.h")]
    if not force and BINDING_OUT.exists():
        t = BINDING_OUT.stat().st_mtime
        if all(p.stat().st_mtime <= t for p in deps):
            return BINDING_OUT
    import sysconfig

    import torch
    root = Path(torch.__file__).resolve().parent
    tmp = BINDING_OUT.with_suffix(".so.tmp")
    cuda = Path(nvcc()).resolve().parent.parent / "include"
    inc = [INCLUDE, root / "include", root / "include/torch/csrc/api/include", cuda,
           sysconfig.get_paths()["include"]]
    cmd = [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-fPIC", "-shared",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
           *[f"-I{p}" for p in inc], str(BINDING), "-o", str(tmp), f"-L{root / 'lib'}",
           "-ltorch_python", "-ltorch_cpu", "-ltorch", "-lc10", "-lc10_cuda"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"{BINDING.name} failed to build:\n{r.stdout}\n{r.stderr}")
    os.replace(tmp, BINDING_OUT)
    return BINDING_OUT


def build(force: bool = False, verbose_ptxas: bool = False) -> Path:
    build_binding(force)
    srcs = sources()
    if not force and not _stale(srcs):
        return OUT
    OBJ_DIR.mkdir(exist_ok=True)
    with cf.ThreadPoolExecutor(max_workers=min(8, len(srcs))) as ex:
        objs = list(ex.map(lambda s: _compile(s, verbose_ptxas), srcs))
    tmp = OUT.with_suffix(".so.tmp")
    cmd = [nvcc(), *ARCH, "-shared", "-cudart", "static", "-o", str(tmp), *map(str, objs)]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"link failed:\n{r.stdout}\n{r.stderr}")
    os.replace(tmp, OUT)
    return OUT


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose_ptxas="--verbose-ptxas" in sys.argv))
