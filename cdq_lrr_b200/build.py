"""Build recipe of libcdq_b200.so, the CUDA/C++ library behind include/cdq.h.

Compiles every source in csrc/ for sm_100a only (no other architecture, no
PTX fallback) with nvcc and links one shared library next to this file, so
the built library travels with the source tree. Objects are cached in
_build/ and rebuilt when a source or header is newer.

The Python module _cdq_torch.*.so beside it (csrc/torch, the direct entry of
the calls whose host time counts) is compiled by the host compiler against the
installed torch's headers and linked to the library. Its name holds the torch
and the Python that it was compiled for. Without torch only the library is
built, which needs nvcc and its host compiler alone.

    python -m cdq_lrr_b200.build          # or: from cdq_lrr_b200.build import build
"""
from __future__ import annotations

import os
import shutil
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

PKG = Path(__file__).resolve().parent
ROOT = PKG.parent
CSRC = PKG / "csrc"
INCLUDE = ROOT / "include"
BUILD = PKG / "_build"
LIB = PKG / "libcdq_b200.so"
TORCH_SRC = CSRC / "torch" / "cdq_torch.cpp"

ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
NVCC_FLAGS = ARCH + ["-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC",
                     "-Xcompiler", "-fvisibility=hidden", "--expt-relaxed-constexpr",
                     f"-I{INCLUDE}", f"-I{CSRC}"]


def _nvcc() -> str:
    cand = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(cand):
        raise RuntimeError("nvcc not found: the CUDA toolkit is required to build libcdq_b200")
    return cand


def _sources() -> list[Path]:
    return sorted(list(CSRC.glob("*.cu")) + list(CSRC.glob("*.cpp")))


def _headers() -> list[Path]:
    return sorted(list(CSRC.glob("*.cuh")) + list(INCLUDE.glob("*.h")))


def _stale(obj: Path, src: Path) -> bool:
    if not obj.exists():
        return True
    t = obj.stat().st_mtime
    return any(p.stat().st_mtime > t for p in [src, *_headers()])


def build(verbose: bool = False, extra: list[str] | None = None) -> Path:
    nvcc = _nvcc()
    BUILD.mkdir(exist_ok=True)
    extra = list(extra or [])
    jobs = []
    for src in _sources():
        obj = BUILD / (src.name + ".o")
        if _stale(obj, src):
            cmd = [nvcc, *NVCC_FLAGS, *extra, "-c", str(src), "-o", str(obj)]
            if src.suffix == ".cpp":
                cmd = [nvcc, "-x", "cu", *NVCC_FLAGS, *extra, "-c", str(src), "-o", str(obj)]
            jobs.append((src, cmd))
    def run(job):
        src, cmd = job
        if verbose:
            print(" ".join(cmd), flush=True)
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"nvcc failed on {src.name}:\n{r.stdout}\n{r.stderr}")
        if verbose and (r.stdout or r.stderr):
            print(r.stdout + r.stderr, flush=True)
    with ThreadPoolExecutor(max_workers=max(1, min(len(jobs), os.cpu_count() or 1))) as ex:
        list(ex.map(run, jobs))
    objs = [str(BUILD / (s.name + ".o")) for s in _sources()]
    if jobs or not LIB.exists() or any(Path(o).stat().st_mtime > LIB.stat().st_mtime for o in objs):
        tmp = LIB.with_suffix(".so.tmp")
        cmd = [nvcc, *ARCH, "-shared", "-o", str(tmp), *objs, "-lcudart"]
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"link failed:\n{r.stdout}\n{r.stderr}")
        os.replace(tmp, LIB)
    build_torch(verbose)
    return LIB


def build_torch(verbose: bool = False) -> Path | None:
    """The Python module over the library (rebuilt when its source or the C header is newer; another torch or Python
    has one of its own). None where torch is not installed: the C library stands alone."""
    import sysconfig

    try:
        import torch
    except ImportError:
        return None

    from ._lib import direct_path
    path = direct_path()
    newest = max(p.stat().st_mtime for p in (TORCH_SRC, INCLUDE / "cdq.h"))
    if path.exists() and path.stat().st_mtime >= newest:
        return path
    from torch.utils import cpp_extension
    cuda = Path(_nvcc()).resolve().parent.parent
    libs = [p for p in cpp_extension.library_paths(device_type="cuda")] + [str(cuda / "lib64")]
    tmp = path.with_suffix(".so.tmp")
    cmd = ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", f"-I{INCLUDE}",
           *[f"-isystem{p}" for p in cpp_extension.include_paths(device_type="cuda")],
           f"-isystem{cuda / 'include'}", f"-isystem{sysconfig.get_paths()['include']}", str(TORCH_SRC), "-o", str(tmp),
           f"-L{PKG}", "-l:libcdq_b200.so", "-Wl,-rpath,$ORIGIN", *[f"-L{p}" for p in libs],
           "-lc10", "-lc10_cuda", "-ltorch", "-ltorch_cpu", "-ltorch_python"]
    if verbose:
        print(" ".join(cmd), flush=True)
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"g++ failed on {TORCH_SRC.name}:\n{r.stdout}\n{r.stderr}")
    os.replace(tmp, path)
    return path


if __name__ == "__main__":
    print(build(verbose="-v" in sys.argv))
