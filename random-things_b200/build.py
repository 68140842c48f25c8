"""Builds libxn_fused.so, the sm_100a fused layer-op library, in-tree, and
xn_torch.so, the part of the Python binding that is a CPython extension.

Usage: python random-things_b200/build.py [--force] [--verbose]

Each csrc/*.cu file is compiled to an object with nvcc for sm_100a only, then
linked into one shared library next to this file. The C ABI it exports is
declared in include/xn_fused.h. Objects are rebuilt when their source or any
header is newer. The binding needs torch and Python's headers; without them the
command builds the library alone, which is all that C, C++ and Rust callers use.
"""
from __future__ import annotations

import argparse
import os
import shutil
import subprocess
import sys
from pathlib import Path

PKG_DIR = Path(__file__).resolve().parent
REPO = PKG_DIR.parent
CSRC = PKG_DIR / "csrc"
INCLUDE = REPO / "include"
BUILD_DIR = PKG_DIR / "_build"
LIB_PATH = PKG_DIR / "libxn_fused.so"
BINDING_PATH = PKG_DIR / "xn_torch.so"

ARCH_FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a"]
# -fmad=false: the reference CPU backend never fuses a*b+c, so neither may the
# kernels (explicit __f*_rn intrinsics are used as well; CUDA's math functions
# use explicit fma internally and are unaffected).
NVCC_FLAGS = [
    "-O3",
    "-std=c++17",
    "-lineinfo",
    "-fmad=false",
    "-Xcompiler",
    "-fPIC",
    "-Xcompiler",
    "-fvisibility=hidden",
    "--expt-relaxed-constexpr",
]


def nvcc_path() -> str:
    cand = os.environ.get("NVCC") or shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not Path(cand).exists():
        raise RuntimeError("nvcc not found; the fused-op library needs the CUDA toolkit to build")
    return cand


def host_compiler() -> list[str]:
    # A gcc wrapper earlier on PATH may lack parts of the toolchain; prefer the system one.
    for c in ("/usr/bin/g++",):
        if Path(c).exists():
            return ["-ccbin", c]
    return []


def sources() -> list[Path]:
    return sorted(CSRC.glob("*.cu"))


def headers() -> list[Path]:
    return sorted(list(CSRC.glob("*.cuh")) + list(CSRC.glob("*.h")) + list(INCLUDE.glob("*.h")))


def _newest(paths: list[Path]) -> float:
    return max((p.stat().st_mtime for p in paths), default=0.0)


def build(force: bool = False, verbose: bool = False, ptxas_verbose: bool = False) -> Path:
    nvcc = nvcc_path()
    BUILD_DIR.mkdir(exist_ok=True)
    hdr_time = _newest(headers())
    objs = []
    for src in sources():
        obj = BUILD_DIR / (src.stem + ".o")
        objs.append(obj)
        if not force and obj.exists() and obj.stat().st_mtime >= max(src.stat().st_mtime, hdr_time):
            continue
        cmd = [nvcc, *host_compiler(), *ARCH_FLAGS, *NVCC_FLAGS, f"-I{INCLUDE}", f"-I{CSRC}",
               "-c", str(src), "-o", str(obj)]
        # The exported C ABI keeps default visibility through XN_API in the sources.
        if ptxas_verbose:
            cmd.insert(-4, "-Xptxas=-v")
        if verbose:
            print(" ".join(cmd), flush=True)
        subprocess.run(cmd, check=True)
    if force or not LIB_PATH.exists() or LIB_PATH.stat().st_mtime < _newest(objs):
        tmp = LIB_PATH.with_suffix(".so.tmp")
        cmd = [nvcc, *host_compiler(), *ARCH_FLAGS, "-shared", "-o", str(tmp), *map(str, objs),
               "-cudart", "static"]
        if verbose:
            print(" ".join(cmd), flush=True)
        subprocess.run(cmd, check=True)
        os.replace(tmp, LIB_PATH)
    return LIB_PATH


def binding_lacks() -> str | None:
    """What the binding cannot be built without here, or None."""
    import importlib.util
    import sysconfig

    if importlib.util.find_spec("torch") is None:
        return "torch is not installed"
    if not (Path(sysconfig.get_paths()["include"]) / "Python.h").exists():
        return "Python's headers are not installed"
    return None


def build_binding(force: bool = False, verbose: bool = False) -> Path:
    """host/xn_torch.cpp against this Python's torch, linked with libxn_fused.so
    next to it. Built again when a source is newer or the torch or Python that
    it was built against is another one."""
    import sysconfig

    import torch
    from torch.utils import cpp_extension

    built_for = "\n".join([sys.version, str(sysconfig.get_config_var("SOABI")), torch.__version__, str(torch.__file__)])
    stamp = BUILD_DIR / (BINDING_PATH.stem + ".built_for")
    src = PKG_DIR / "host" / "xn_torch.cpp"
    newest = max(src.stat().st_mtime, (INCLUDE / "xn_fused.h").stat().st_mtime, LIB_PATH.stat().st_mtime)
    same = stamp.exists() and stamp.read_text() == built_for
    if not force and same and BINDING_PATH.exists() and BINDING_PATH.stat().st_mtime >= newest:
        return BINDING_PATH
    cxx = host_compiler()[1:] or ["g++"]
    inc = [f"-I{p}" for p in (INCLUDE, sysconfig.get_paths()["include"], *cpp_extension.include_paths(device_type="cuda"))]
    lib = [f"-L{p}" for p in cpp_extension.library_paths(device_type="cuda")]
    tmp = BINDING_PATH.with_suffix(".so.tmp")
    cmd = [*cxx, "-O2", "-std=c++17", "-shared", "-fPIC", "-fvisibility=hidden", "-DTORCH_EXTENSION_NAME=xn_torch", *inc, str(src),
           "-o", str(tmp), f"-L{PKG_DIR}", "-lxn_fused", "-Wl,-rpath,$ORIGIN", *lib, "-lc10", "-lc10_cuda", "-ltorch_cpu",
           "-ltorch_python"]
    if verbose:
        print(" ".join(cmd), flush=True)
    subprocess.run(cmd, check=True)
    os.replace(tmp, BINDING_PATH)
    BUILD_DIR.mkdir(exist_ok=True)
    stamp.write_text(built_for)
    return BINDING_PATH


def main(argv: list[str] | None = None) -> int:
    ap = argparse.ArgumentParser(description=__doc__)
    ap.add_argument("--force", action="store_true")
    ap.add_argument("--verbose", action="store_true")
    ap.add_argument("--ptxas-verbose", action="store_true", help="print registers / spills per kernel")
    a = ap.parse_args(argv)
    path = build(force=a.force, verbose=a.verbose, ptxas_verbose=a.ptxas_verbose)
    print(path)
    lacks = binding_lacks()
    if lacks is None:
        print(build_binding(force=a.force, verbose=a.verbose))
    else:
        print(f"{BINDING_PATH.name}, the Python binding, is not built: {lacks}", file=sys.stderr)
    return 0


if __name__ == "__main__":
    sys.exit(main())
