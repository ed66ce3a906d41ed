"""Build the sm_100a C-ABI library in-tree (``logitfill_b200/_lib/``).

    python -m logitfill_b200.build                 # or __graft_entry__.build()
    python logitfill_b200/build.py --library       # the C library alone: needs no torch

nvcc cross-compiles for B200 without a GPU.  The shared library links the
CUDA runtime statically and exports only the ``lf_*`` symbols declared in
``include/logitfill_b200.h``.  The compiled Python binding of the 4-bit cache
(``csrc/int4_binding.cpp``, against the installed torch) lies next to it.
"""
from __future__ import annotations

import os
import shutil
import subprocess
import sys
from pathlib import Path

PKG = Path(__file__).resolve().parent
ROOT = PKG.parent
CSRC = PKG / "csrc"
OUT_DIR = PKG / "_lib"
LIB_NAME = "liblogitfill_b200.so"
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]


def nvcc() -> str:
    found = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not Path(found).exists():
        raise RuntimeError("nvcc not found; the CUDA 12.9 toolkit is required to build logitfill_b200")
    return found


def sources() -> list[Path]:
    return sorted(CSRC.glob("*.cu"))


def binding_path() -> Path:
    """The binding for this Python and this torch, whose C++ classes it is compiled
    against: both are in the name."""
    import sysconfig

    import torch

    return OUT_DIR / f"int4_binding.torch-{torch.__version__}.{sysconfig.get_config_var('SOABI')}.so"


def build_binding(verbose: bool = False, force: bool = False) -> Path:
    """g++ of the 4-bit cache's Python binding, linked to torch and the library."""
    src, out, lib = CSRC / "int4_binding.cpp", binding_path(), OUT_DIR / LIB_NAME
    deps = (src, ROOT / "include" / "logitfill_b200.h", Path(__file__))
    if not force and out.exists() and all(out.stat().st_mtime >= d.stat().st_mtime for d in deps):
        return out
    import sysconfig

    import torch

    torch_dir = Path(torch.__file__).resolve().parent
    cuda = Path(nvcc()).resolve().parents[1] / "include"
    tmp = out.with_suffix(".so.tmp")
    cmd = ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", "-I", str(ROOT / "include"),
           "-isystem", str(torch_dir / "include"), "-isystem", str(torch_dir / "include" / "torch" / "csrc" / "api" / "include"),
           "-isystem", str(cuda), "-isystem", sysconfig.get_path("include"), str(src), "-o", str(tmp),
           str(lib), "-L", str(torch_dir / "lib"), "-ltorch_python", "-ltorch_cpu", "-lc10", "-lc10_cuda",
           "-Wl,-rpath,$ORIGIN"]
    if verbose:
        print(" ".join(cmd), flush=True)
    done = subprocess.run(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)
    if done.returncode != 0:
        raise RuntimeError(f"g++ failed on {src.name}:\n{done.stdout}")
    os.replace(tmp, out)
    return out


def build(verbose: bool = False, force: bool = False) -> Path:
    """Build the library and the binding; returns the library's path."""
    out = build_library(verbose, force)
    build_binding(verbose, force)
    return out


def build_library(verbose: bool = False, force: bool = False) -> Path:
    """Build the C library, which needs nvcc and its host compiler only."""
    OUT_DIR.mkdir(exist_ok=True)
    out = OUT_DIR / LIB_NAME
    srcs = sources()
    deps = srcs + sorted(CSRC.glob("*.cuh")) + [ROOT / "include" / "logitfill_b200.h", Path(__file__)]
    if not force and out.exists() and all(out.stat().st_mtime >= d.stat().st_mtime for d in deps):
        return out
    build_dir = OUT_DIR / "obj"
    build_dir.mkdir(exist_ok=True)
    common = [nvcc(), *ARCH, "-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC,-fvisibility=hidden",
              "-I", str(ROOT / "include"), "-I", str(CSRC), "--expt-relaxed-constexpr"]
    objs = []
    procs = []
    for src in srcs:
        obj = build_dir / (src.stem + ".o")
        cmd = common + ["-c", str(src), "-o", str(obj)]
        if verbose:
            print(" ".join(cmd), flush=True)
        procs.append((src, subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT)))
        objs.append(obj)
    failed = []
    for src, proc in procs:
        log = proc.communicate()[0].decode()
        if proc.returncode != 0:
            failed.append(f"{src.name}:\n{log}")
        elif verbose and log.strip():
            print(log)
    if failed:
        raise RuntimeError("nvcc failed:\n" + "\n".join(failed))
    tmp = out.with_suffix(".so.tmp")
    link = [nvcc(), *ARCH, "-shared", "-o", str(tmp), "-Xlinker", f"-soname={LIB_NAME}", *map(str, objs), "-cudart", "static"]
    if verbose:
        print(" ".join(link), flush=True)
    subprocess.run(link, check=True)
    os.replace(tmp, out)
    return out


if __name__ == "__main__":
    make = build_library if "--library" in sys.argv else build
    print(make(verbose="-v" in sys.argv, force="-f" in sys.argv))
