"""Build libdequant_b200.so in-tree (sm_100a only).

    python -m dequant_project_b200.build [--force] [--verbose-ptxas]

Each ``csrc/*.cu`` is compiled by nvcc for ``arch=compute_100a,code=sm_100a``
with ``-lineinfo`` and linked into ``dequant_project_b200/libdequant_b200.so``
next to this file (static CUDA runtime, no torch dependency). The shared
library is the product's C ABI (include/dequant_b200.h); the Python package
loads it with ctypes. The paged-cache operators' calls are also bound natively
(``binding/paged_binding.cpp``, built against the installed torch into
``_paged_binding.so``; left out, with a note, where torch, a C++ compiler or
Python's headers are missing).
"""

from __future__ import annotations

import concurrent.futures as cf
import json
import os
import shutil
import subprocess
import sys
import sysconfig
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


def _binding_command(torch, out: Path) -> list[str]:
    root = Path(torch.__file__).resolve().parent
    cuda = Path(nvcc()).resolve().parent.parent / "include"
    inc = [INCLUDE, root / "include", root / "include/torch/csrc/api/include", cuda,
           sysconfig.get_paths()["include"]]
    return [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-fPIC", "-shared",
            f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
            f'-DDQG_BUILT_FOR="{torch.__version__}"',
            *[f"-I{p}" for p in inc], str(BINDING), "-o", str(out), f"-L{root / 'lib'}",
            "-ltorch_python", "-ltorch_cpu", "-ltorch", "-lc10", "-lc10_cuda"]


def build_binding(force: bool = False) -> Path | None:
    """The native binding of the paged operators (g++, torch's headers), built
    again when its sources, torch, the interpreter or the command change. None
    where torch, a compiler or Python's headers are missing: the C library does
    without."""
    try:
        import torch
    except ImportError as exc:
        return _no_binding(f"torch cannot be imported ({exc})")
    if shutil.which(os.environ.get("CXX", "g++")) is None:
        return _no_binding("no C++ compiler (g++, or CXX)")
    if not (Path(sysconfig.get_paths()["include"]) / "Python.h").exists():
        return _no_binding("Python.h is missing")
    tmp = BINDING_OUT.with_suffix(".so.tmp")
    cmd = _binding_command(torch, tmp)
    built = json.dumps([cmd, torch.__version__, sys.version, sysconfig.get_config_var("SOABI")])
    stamp = OBJ_DIR / "paged_binding.json"
    deps = [BINDING, *INCLUDE.glob("*.h")]
    if (not force and BINDING_OUT.exists() and stamp.exists() and stamp.read_text() == built
            and all(p.stat().st_mtime <= BINDING_OUT.stat().st_mtime for p in deps)):
        return BINDING_OUT
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"{BINDING.name} failed to build:\n{r.stdout}\n{r.stderr}")
    OBJ_DIR.mkdir(exist_ok=True)
    os.replace(tmp, BINDING_OUT)
    stamp.write_text(built)
    return BINDING_OUT


def _no_binding(why: str) -> None:
    print(f"the paged operators' binding is not built: {why}", file=sys.stderr)


def build(force: bool = False, verbose_ptxas: bool = False) -> Path:
    """The C library, and after it the binding, which needs torch."""
    _build_library(force, verbose_ptxas)
    build_binding(force)
    return OUT


def _build_library(force: bool, verbose_ptxas: bool) -> None:
    srcs = sources()
    if not force and not _stale(srcs):
        return
    OBJ_DIR.mkdir(exist_ok=True)
    with cf.ThreadPoolExecutor(max_workers=min(8, len(srcs))) as ex:
        objs = list(ex.map(lambda s: _compile(s, verbose_ptxas), srcs))
    tmp = OUT.with_suffix(".so.tmp")
    cmd = [nvcc(), *ARCH, "-shared", "-cudart", "static", "-o", str(tmp), *map(str, objs)]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"link failed:\n{r.stdout}\n{r.stderr}")
    os.replace(tmp, OUT)


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose_ptxas="--verbose-ptxas" in sys.argv))
