"""Builds nestquant_b200/libnestquant_b200.so in-tree with nvcc for sm_100a (no GPU needed to compile).

    python -m nestquant_b200.build [--force] [--verbose]

Replaces the reference's JIT build (sm120/build.py:7-12): same idea (one shared object holding every kernel of the
MoE layer path), but ahead of time, with a plain C ABI instead of a torch extension module.
"""
import concurrent.futures as cf
import os
import shutil
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
OBJ = os.path.join(HERE, "build")
LIB = os.path.join(HERE, "libnestquant_b200.so")
OPS = os.path.join(HERE, "_torch_ops.so")
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
FLAGS = ["-O3", "-std=c++17", "-lineinfo", "-Xcompiler", "-fPIC", "--expt-relaxed-constexpr", "-Xptxas", "-v"]


def nvcc():
    for c in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if c and os.path.exists(c):
            return c
    raise RuntimeError("nvcc not found (set NVCC)")


def _torch_ops(lib, force=False, verbose=False):
    """nestquant_b200/_torch_ops.so, the torch side of routing.py and w4.py (host code only), linked against the library.  Where there is no torch the
    library stands alone, for hosts that call its C entry points."""
    src = os.path.join(CSRC, "torch_ops.cpp")
    fresh = os.path.exists(OPS) and os.path.getmtime(OPS) >= max(os.path.getmtime(f) for f in (src, os.path.join(os.path.dirname(HERE), "include", "nestquant_b200.h")))
    if fresh and not force:
        return OPS
    import sysconfig
    try:
        import torch
        from torch.utils import cpp_extension as X
    except ImportError as e:
        if os.path.exists(OPS) and not fresh:
            os.remove(OPS)          # (older than its source or the header: not beside a newer library)
        print(f"{OPS} is not built, routing.py and w4.py need it: no torch here ({e})", file=sys.stderr)
        return None
    inc = X.include_paths("cuda") + [sysconfig.get_paths()["include"]]
    libs = X.library_paths("cuda")
    cmd = ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", "-DTORCH_EXTENSION_NAME=_torch_ops"]
    cmd += [f"-isystem{d}" for d in inc] + [src, "-o", OPS] + [f"-L{d}" for d in libs] + [f"-L{HERE}", "-l:" + os.path.basename(lib), "-Wl,-rpath,$ORIGIN"]
    cmd += ["-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch", "-ltorch_python", "-lcudart"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if verbose:
        print(r.stderr, file=sys.stderr)
    if r.returncode:
        raise RuntimeError("g++ failed for torch_ops.cpp:\n" + r.stderr[-4000:])
    return OPS


def sources():
    return sorted(f for f in os.listdir(CSRC) if f.endswith(".cu"))


def _newest_dep():
    t = 0.0
    for d in (CSRC, os.path.join(os.path.dirname(HERE), "include")):
        for f in os.listdir(d):
            t = max(t, os.path.getmtime(os.path.join(d, f)))
    return t


def _compile(src, verbose):
    obj = os.path.join(OBJ, src[:-3] + ".o")
    defs = ["-D" + d for d in os.environ.get("NQ_DEFS", "").split(",") if d]     # e.g. NQ_DEFS=NQ_GEMV_CODES=0x81
    cmd = [nvcc()] + ARCH + FLAGS + defs + ["-c", os.path.join(CSRC, src), "-o", obj]
    r = subprocess.run(cmd, capture_output=True, text=True)
    with open(obj[:-2] + ".ptxas.log", "w") as f:       # registers / spills / shared memory per kernel
        f.write(r.stderr)
    if r.returncode:
        raise RuntimeError(f"nvcc failed for {src}:\n{r.stderr[-4000:]}")
    if verbose:
        print(r.stderr, file=sys.stderr)
    return obj


def build(force=False, verbose=False):
    """Compile every csrc/*.cu and link the shared library, and, where there is torch, the torch module on top of it.  Returns the library's path."""
    os.makedirs(OBJ, exist_ok=True)
    if not force and os.path.exists(LIB) and os.path.getmtime(LIB) >= _newest_dep():
        _torch_ops(LIB, force, verbose)
        return LIB
    with cf.ThreadPoolExecutor(max_workers=min(8, os.cpu_count() or 1)) as ex:
        objs = list(ex.map(lambda s: _compile(s, verbose), sources()))
    r = subprocess.run([nvcc()] + ARCH + ["-shared", "-o", LIB] + objs + ["-lcudart"], capture_output=True, text=True)
    if r.returncode:
        raise RuntimeError("link failed:\n" + r.stderr[-4000:])
    _torch_ops(LIB, force, verbose)
    return LIB


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="--verbose" in sys.argv))
