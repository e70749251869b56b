"""Build the sm_100a CUDA library ``libb200moe.so`` and the torch binding of its stateless
operators, ``b200moe_ops.so``, in place (next to this file).

Each ``csrc/*.cu`` is compiled with nvcc for ``-gencode arch=compute_100a,code=sm_100a``
into an object, then linked into one shared library that the ctypes front end
loads.  Objects are rebuilt only when a source or header is newer.
"""

from __future__ import annotations

import hashlib
import os
import subprocess
import sys
import sysconfig
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

HERE = Path(__file__).resolve().parent
CSRC = HERE / "csrc"
OBJ = HERE / "_build"
LIB = HERE / "libb200moe.so"
OPS = HERE / "b200moe_ops.so"
INCLUDE = HERE.parent / "include"
NVCC = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
FLAGS = ["-O3", "-std=c++17", "-lineinfo", "-Xcompiler", "-fPIC", "-I", str(INCLUDE), "--expt-relaxed-constexpr"]


def _newest_header() -> float:
    hs = list(CSRC.glob("*.cuh")) + list(CSRC.glob("*.h")) + list(INCLUDE.glob("*.h"))
    return max(h.stat().st_mtime for h in hs)


def _compile(src: Path, verbose: bool) -> Path:
    obj = OBJ / (src.stem + ".o")
    if obj.exists() and obj.stat().st_mtime >= max(src.stat().st_mtime, _newest_header()):
        return obj
    cmd = [NVCC, *ARCH, *FLAGS, "-c", str(src), "-o", str(obj)]
    if verbose:
        cmd.insert(1, "-Xptxas=-v")
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"nvcc failed on {src.name}:\n{r.stdout}\n{r.stderr}")
    if verbose:
        sys.stderr.write(r.stderr)
    return obj


def _pin(lib: Path) -> None:
    """The digest the loader checks a library against (a different file is refused)."""
    lib.with_suffix(".so.sha256").write_text(hashlib.sha256(lib.read_bytes()).hexdigest() + "\n")


def _build_ops() -> None:
    """``csrc/bind.cpp``: the torch binding of the stateless operators, linked to the library beside it."""
    import torch

    src = CSRC / "bind.cpp"
    newest = max(src.stat().st_mtime, *(h.stat().st_mtime for h in INCLUDE.glob("*.h")))
    if not OPS.exists() or OPS.stat().st_mtime < newest:
        t = Path(torch.__file__).parent
        cmd = ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
               "-I", str(t / "include"), "-I", str(t / "include/torch/csrc/api/include"),
               "-I", str(Path(NVCC).parent.parent / "include"), "-I", sysconfig.get_paths()["include"], str(src),
               "-o", str(OPS), "-L", str(HERE), "-l:" + LIB.name, "-L", str(t / "lib"), "-lc10", "-lc10_cuda",
               "-ltorch_cpu", "-ltorch_cuda", "-ltorch", "-ltorch_python", "-Wl,-rpath,$ORIGIN",
               f"-Wl,-rpath,{t / 'lib'}"]
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"g++ failed on {src.name}:\n{r.stdout}\n{r.stderr}")
    _pin(OPS)


def build(verbose: bool = False) -> Path:
    OBJ.mkdir(exist_ok=True)
    srcs = sorted(CSRC.glob("*.cu"))
    with ThreadPoolExecutor(max_workers=min(8, len(srcs))) as ex:
        objs = list(ex.map(lambda s: _compile(s, verbose), srcs))
    if not LIB.exists() or LIB.stat().st_mtime < max(o.stat().st_mtime for o in objs):
        cmd = [NVCC, *ARCH, "-shared", "-o", str(LIB), *map(str, objs), "-lcudart"]
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"link failed:\n{r.stdout}\n{r.stderr}")
    _pin(LIB)
    _build_ops()
    return LIB


if __name__ == "__main__":
    print(build(verbose="-v" in sys.argv))
