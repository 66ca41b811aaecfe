"""Build libcutetts_b200.so (sm_100a) in-tree with nvcc, and the torch binding
of the paged operators beside it.  The library needs the CUDA toolkit alone;
where torch with CUDA, or Python's headers, are missing it is built without
the binding.

Each source compiles to an object under rcutetts_b200/_build/ (in parallel,
skipped when up to date), then one shared library is linked next to this
file.  The CUDA runtime is linked statically so the library does not depend
on the runtime version torch ships.
"""
from __future__ import annotations

import concurrent.futures as cf
import os
import shutil
import subprocess
import sys
import sysconfig

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
CSRC = os.path.join(HERE, "csrc")
BUILD = os.path.join(HERE, "_build")
LIB = os.path.join(HERE, "libcutetts_b200.so")

ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
# the torch binding of the paged operators (rcutetts_b200/paged.py)
EXT_SRC = os.path.join(HERE, "csrc_py", "paged_ext.cpp")
EXT = os.path.join(HERE, "_paged_ext.so")
NVFLAGS = ["-O3", "-std=c++17", "-lineinfo", "--expt-relaxed-constexpr", "-Xcompiler", "-fPIC",
           "-Xcompiler", "-fvisibility=hidden", "-I", os.path.join(ROOT, "include")]


def nvcc() -> str:
    p = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(p):
        raise RuntimeError("nvcc not found")
    return p


def sources():
    out = []
    for f in sorted(os.listdir(CSRC)):
        if f.endswith(".cu") or f.endswith(".cpp"):
            out.append(os.path.join(CSRC, f))
    return out


def _deps_mtime() -> float:
    m = 0.0
    for d in (CSRC, os.path.join(ROOT, "include")):
        for f in os.listdir(d):
            if f.endswith((".h", ".cuh")):
                m = max(m, os.path.getmtime(os.path.join(d, f)))
    return m


def _compile(src: str, hdr_mtime: float, verbose: bool) -> str:
    obj = os.path.join(BUILD, os.path.basename(src) + ".o")
    if os.path.exists(obj) and os.path.getmtime(obj) >= max(os.path.getmtime(src), hdr_mtime):
        return obj
    cmd = [nvcc()] + ARCH + NVFLAGS + ["-c", src, "-o", obj]
    if src.endswith(".cpp"):
        cmd = [nvcc(), "-x", "cu"] + ARCH + NVFLAGS + ["-c", src, "-o", obj]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"nvcc failed for {src}:\n{r.stderr}")
    if verbose and r.stderr.strip():
        print(r.stderr, file=sys.stderr)
    return obj


def build(verbose: bool = False) -> str:
    os.makedirs(BUILD, exist_ok=True)
    hdr = _deps_mtime()
    srcs = sources()
    with cf.ThreadPoolExecutor(max_workers=min(8, os.cpu_count() or 4)) as ex:
        objs = list(ex.map(lambda s: _compile(s, hdr, verbose), srcs))
    if not os.path.exists(LIB) or os.path.getmtime(LIB) < max(os.path.getmtime(o) for o in objs):
        cmd = [nvcc()] + ARCH + ["-shared", "-o", LIB] + objs + ["-cudart", "static", "-lcuda"]
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"link failed:\n{r.stderr}")
    build_ext()
    return LIB


def _no_ext(why: str) -> None:
    print(f"the torch binding of the paged operators is not built: {why}", file=sys.stderr)


def build_ext() -> str | None:
    """_paged_ext.so against the installed torch, linked to the library beside it; again when its source, torch or Python is another.
    None, and a word on stderr, where there is no torch to build it against."""
    try:
        import torch
    except (ImportError, OSError) as e:  # (OSError: one of its libraries is missing)
        return _no_ext(str(e))
    newest = max(os.path.getmtime(p) for p in (EXT_SRC, os.path.join(ROOT, "include", "cutetts_b200.h")))
    made_for, stamp = f"torch {torch.__version__}, {sysconfig.get_config_var('SOABI')}", os.path.join(BUILD, "paged_ext.made_for")
    if os.path.exists(EXT) and os.path.getmtime(EXT) >= newest and os.path.exists(stamp):
        with open(stamp) as f:
            if f.read() == made_for:
                return EXT
    troot = os.path.dirname(torch.__file__)
    for p in (os.path.join(troot, "lib", "libtorch_cuda.so"), os.path.join(troot, "include", "ATen", "ATen.h"),
              os.path.join(sysconfig.get_paths()["include"], "Python.h")):
        if not os.path.exists(p):
            return _no_ext(f"{p} is missing")
    inc = [os.path.join(troot, "include"), os.path.join(troot, "include", "torch", "csrc", "api", "include"),
           os.path.join(os.path.dirname(os.path.dirname(nvcc())), "include"), sysconfig.get_paths()["include"]]
    cmd = [shutil.which("g++") or "g++", "-O2", "-std=c++17", "-shared", "-fPIC", "-fvisibility=hidden",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", f'-DPAGED_EXT_TORCH="{torch.__version__}"']
    cmd += [f"-I{p}" for p in inc] + [EXT_SRC, "-o", EXT + ".new", f"-L{HERE}", "-l:libcutetts_b200.so", f"-L{os.path.join(troot, 'lib')}",
                                      "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch_cuda", "-ltorch_python", "-Wl,-rpath,$ORIGIN"]
    os.makedirs(BUILD, exist_ok=True)
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"g++ failed for {EXT_SRC}:\n{r.stderr[-4000:]}")
    os.replace(EXT + ".new", EXT)  # (a process may have the old one mapped)
    with open(stamp, "w") as f:
        f.write(made_for)
    return EXT


if __name__ == "__main__":
    print(build(verbose="-v" in sys.argv))
