"""Builds libwebgllm_b200.so, the library behind include/webgllm_q4.h.

Plain nvcc, sm_100a only (B200), into the package directory so that the
shared object ships with the source tree. Run as ``python -m
webgllm_b200.build`` or through ``__graft_entry__.build()``.
"""
from __future__ import annotations

import os
import shutil
import subprocess
import sys
import sysconfig
from pathlib import Path

PKG = Path(__file__).resolve().parent
ROOT = PKG.parent
CSRC = PKG / "csrc"
LIB = PKG / "libwebgllm_b200.so"
HOST = PKG / "_host.so"
OBJ_DIR = PKG / "_build"

ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
NVCC_FLAGS = [
    "-O3", "-std=c++17", "-lineinfo", "-Xcompiler", "-fPIC",
    "--expt-relaxed-constexpr", "-Xptxas", "-warn-spills",
]


def nvcc() -> str:
    cuda = os.environ.get("CUDA_HOME", "/usr/local/cuda")
    path = Path(cuda) / "bin" / "nvcc"
    return str(path) if path.exists() else (shutil.which("nvcc") or "nvcc")


def sources() -> list[Path]:
    return sorted(CSRC.glob("*.cu"))


def _stale(target: Path, deps: list[Path]) -> bool:
    if not target.exists():
        return True
    t = target.stat().st_mtime
    return any(d.stat().st_mtime > t for d in deps)


def host_target() -> str:
    """What _host.so is compiled against: it is used with nothing else."""
    import torch

    return f"{torch.__version__} {sys.version_info[0]}.{sys.version_info[1]}"


def build_host(verbose: bool = False) -> Path | None:
    """Compile csrc/host/ into the Python module _host.so against the installed
    torch. None (and a line on stderr, and no module) where that cannot be done -
    no torch, one without CUDA, no headers, no compiler: the calls then go
    through Python's code."""
    srcs = sorted((CSRC / "host").glob("*.cpp"))
    stamp = OBJ_DIR / "host_torch"
    try:
        import torch
        from torch.utils.cpp_extension import CUDA_HOME, include_paths, library_paths

        target = host_target()
        built_for = stamp.read_text() if stamp.exists() else ""
        if built_for == target and not _stale(HOST, [*srcs, *(ROOT / "include").glob("*.h")]):
            return HOST
        includes = [*include_paths(), sysconfig.get_paths()["include"],
                    str(Path(CUDA_HOME or "/usr/local/cuda") / "include")]
        made = OBJ_DIR / HOST.name
        cmd = [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-fPIC", "-shared",
               f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", f'-DWG_HOST_TARGET="{target}"',
               *(f"-I{i}" for i in includes), *map(str, srcs), "-o", str(made),
               *(f for p in library_paths() for f in (f"-L{p}", f"-Wl,-rpath,{p}")),
               "-ltorch_python", "-ltorch_cpu", "-lc10", "-lc10_cuda"]
        if verbose:
            print(" ".join(cmd), file=sys.stderr)
        subprocess.run(cmd, check=True)
        made.replace(HOST)
    except (ImportError, OSError, subprocess.CalledProcessError) as e:
        HOST.unlink(missing_ok=True)  # (one of another build or torch)
        print(f"{HOST.name} not built: {e}", file=sys.stderr)
        return None
    stamp.write_text(target)
    return HOST


def build(verbose: bool = False, ptxas_info: bool = False) -> Path:
    """Compile every .cu under csrc/ and link the shared library (rebuilds
    only what changed; any header change rebuilds everything), and the module
    of host calls."""
    OBJ_DIR.mkdir(exist_ok=True)
    headers = list(CSRC.glob("*.cuh")) + list((ROOT / "include").glob("*.h"))
    objs = []
    for src in sources():
        obj = OBJ_DIR / (src.stem + ".o")
        objs.append(obj)
        if not _stale(obj, [src, *headers]) and not ptxas_info:
            continue
        cmd = [nvcc(), *ARCH, *NVCC_FLAGS, "-I", str(ROOT / "include"), "-c", str(src), "-o", str(obj)]
        if ptxas_info:
            cmd += ["-Xptxas", "-v"]
        if verbose:
            print(" ".join(cmd), file=sys.stderr)
        subprocess.run(cmd, check=True)
    if _stale(LIB, objs):
        cmd = [nvcc(), *ARCH, "-shared", "-cudart", "static", "-o", str(LIB), *map(str, objs), "-ldl"]
        if verbose:
            print(" ".join(cmd), file=sys.stderr)
        subprocess.run(cmd, check=True)
    build_host(verbose)
    return LIB


if __name__ == "__main__":
    build(verbose=True, ptxas_info="-v" in sys.argv)
    print(LIB)
