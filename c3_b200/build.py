"""Builds libc3cu.so in-tree: every CUDA translation unit for sm_100a plus the C++ host
mirror of the C3 API, linked with the static CUDA runtime so that the library loads on
machines without a GPU driver (calls then report C3CU_ERR_UNSUPPORTED); and _fast_calls.<torch>.so, the
binding of the 8-bit path's calls against the C++ headers of the torch that is installed (csrc/torch).
The binding only shortens a call's time on the host: where it cannot be built, the calls go through
ctypes."""
from __future__ import annotations

import concurrent.futures as cf
import hashlib
import os
import re
import shutil
import subprocess
import sys
import sysconfig
import warnings
from pathlib import Path

PKG = Path(__file__).resolve().parent
ROOT = PKG.parent
CSRC = PKG / "csrc"
HOST = CSRC / "host"
OUT_DIR = PKG / "_build"
LIB = PKG / "libc3cu.so"

NVCC = os.environ.get("NVCC", shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc")
GENCODE = ["-gencode", "arch=compute_100a,code=sm_100a"]
CU_FLAGS = ["-std=c++17", "-O3", "-lineinfo", "-Xcompiler", "-fPIC", "-Xcompiler", "-Wall",
            f"-I{ROOT / 'include'}", f"-I{CSRC}", f"-I{HOST}"] + GENCODE
CXX_FLAGS = ["-std=c++17", "-O2", "-fPIC", "-Wall", "-Wextra", f"-I{ROOT / 'include'}",
             f"-I{HOST}", "-I/usr/local/cuda/include", "-pthread"]


def _sources():
    cu = sorted(CSRC.glob("*.cu"))
    cpp = sorted(CSRC.glob("*.cpp")) + (sorted(HOST.rglob("*.cpp")) if HOST.exists() else [])
    return cu, cpp


def _stale(obj: Path, src: Path) -> bool:
    if not obj.exists():
        return True
    deps = [src] + list(CSRC.glob("*.cuh")) + list(CSRC.glob("*.h")) + \
        list((ROOT / "include").glob("*.h")) + list(HOST.rglob("*.h"))
    t = obj.stat().st_mtime
    return any(d.stat().st_mtime > t for d in deps)


def _compile(src: Path) -> Path:
    rel = src.relative_to(PKG).as_posix().replace("/", "_")
    obj = OUT_DIR / (rel + ".o")
    if not _stale(obj, src):
        return obj
    if src.suffix == ".cu":
        cmd = [NVCC] + CU_FLAGS + ["-c", str(src), "-o", str(obj)]
    else:
        cmd = [os.environ.get("CXX", "g++")] + CXX_FLAGS + ["-c", str(src), "-o", str(obj)]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"compile failed: {' '.join(cmd)}\n{r.stdout}\n{r.stderr}")
    return obj


def _fast_calls_sources() -> tuple[Path, Path]:
    return CSRC / "torch" / "fast_calls.cpp", ROOT / "include" / "c3cu.h"


def fast_calls_path() -> Path:
    """The binding's file, named for the torch and the Python that it is compiled against and for what it is
    compiled from: another torch's classes are laid out differently, and another c3cu.h may declare other
    arguments, so that a binding of theirs must not be loaded."""
    import torch
    tag = re.sub(r"[^0-9A-Za-z]+", "_", f"torch{torch.__version__}_{sys.implementation.cache_tag}")
    text = hashlib.sha256(b"".join(f.read_bytes() for f in _fast_calls_sources())).hexdigest()
    return PKG / f"_fast_calls.{tag}.{text[:12]}.so"


def build_fast_calls() -> Path:
    import torch
    out = fast_calls_path()
    if out.exists():
        return out
    src = _fast_calls_sources()[0]
    home = Path(torch.__file__).resolve().parent
    tmp = out.with_suffix(f".{os.getpid()}.tmp")
    cmd = [os.environ.get("CXX", "g++"), "-std=c++17", "-O2", "-fPIC", "-shared", "-Wall",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", f"-I{ROOT / 'include'}",
           f"-isystem{home / 'include'}", f"-isystem{home / 'include/torch/csrc/api/include'}",
           "-isystem/usr/local/cuda/include", f"-isystem{sysconfig.get_paths()['include']}", str(src), "-o", str(tmp),
           f"-L{home / 'lib'}", "-ltorch_python", "-ltorch_cuda", "-ltorch_cpu", "-ltorch", "-lc10_cuda", "-lc10"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"compile failed: {' '.join(cmd)}\n{r.stdout}\n{r.stderr}")
    os.replace(tmp, out)
    for old in PKG.glob("_fast_calls*.so"):
        if old.name == "_fast_calls.so" or (old != out and old.name.split(".")[1] == out.name.split(".")[1]):
            old.unlink(missing_ok=True)  # from other sources
    return out


def try_build_fast_calls() -> Path | None:
    """None, with a warning, where the binding cannot be built (no C++ compiler, a torch without its headers
    or of another making)."""
    try:
        return build_fast_calls()
    except Exception as e:
        warnings.warn(f"the C++ binding of the 8-bit calls was not built, they go through ctypes: {str(e)[-600:]}",
                      RuntimeWarning, stacklevel=2)
        return None


def build(verbose: bool = False) -> Path:
    OUT_DIR.mkdir(exist_ok=True)
    cu, cpp = _sources()
    with cf.ThreadPoolExecutor(max_workers=os.cpu_count() or 4) as ex:
        fast = ex.submit(try_build_fast_calls)
        objs = list(ex.map(_compile, cu + cpp))
        fast.result()
    if LIB.exists() and all(LIB.stat().st_mtime >= o.stat().st_mtime for o in objs):
        return LIB
    cmd = [NVCC, "-shared", "-cudart", "static", "-o", str(LIB)] + [str(o) for o in objs] + \
        GENCODE + ["-Xlinker", "--no-undefined", "-lpthread", "-ldl", "-lrt"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"link failed: {' '.join(cmd)}\n{r.stdout}\n{r.stderr}")
    if verbose:
        print(f"built {LIB}")
    return LIB


if __name__ == "__main__":
    build(verbose=True)
    sys.exit(0)
