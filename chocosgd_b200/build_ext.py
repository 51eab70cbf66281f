"""Build the in-tree native library ``chocosgd_b200/lib/libchoco_b200.so``.

All CUDA sources are compiled for sm_100a only
(``nvcc -gencode arch=compute_100a,code=sm_100a -lineinfo``); nvcc cross-compiles without
a GPU.  The kernels expose a plain C ABI (raw pointers + ``cudaStream_t``) and are bound
with ctypes (``ops/_lib.py``); one host-only file, the autograd nodes of ``csrc/autograd.cpp``,
is compiled against PyTorch's headers into ``lib/_choco_autograd.so``, which links to the library.
Usage: ``python -m chocosgd_b200.build_ext [--force] [--verbose]``."""
from __future__ import annotations

import hashlib
import os
import shutil
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
SRC = os.path.join(HERE, "csrc")
OUT_DIR = os.path.join(HERE, "lib")
OBJ_DIR = os.path.join(OUT_DIR, "obj")
LIB = os.path.join(OUT_DIR, "libchoco_b200.so")
NODES = os.path.join(OUT_DIR, "_choco_autograd.so")
NODES_SRC = "autograd.cpp"

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a", "-lineinfo", "-O3", "-std=c++17",
    "--use_fast_math" if False else "-DCHOCO_NO_FAST_MATH", "-Xcompiler", "-fPIC", "-Xptxas", "-v",
]
CXX_FLAGS = ["-O3", "-std=c++17", "-fPIC", "-fopenmp"]


def nvcc_path():
    for c in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if c and os.path.exists(c):
            return c
    return None


def sources():
    cu = sorted(f for f in os.listdir(SRC) if f.endswith(".cu"))
    cpp = sorted(f for f in os.listdir(SRC) if f.endswith(".cpp") and f != NODES_SRC)
    return cu, cpp


def _digest():
    h = hashlib.sha256()
    for f in sorted(os.listdir(SRC)):
        if f.endswith((".cu", ".cuh", ".cpp", ".h")):
            with open(os.path.join(SRC, f), "rb") as fh:
                h.update(f.encode())
                h.update(fh.read())
    h.update(" ".join(NVCC_FLAGS).encode())
    import torch

    h.update(torch.__version__.encode())
    return h.hexdigest()


def is_current():
    stamp = os.path.join(OUT_DIR, "build.stamp")
    return os.path.exists(LIB) and os.path.exists(NODES) and os.path.exists(stamp) and open(stamp).read().strip() == _digest()


def _run(cmd, what):
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"{what} failed:\n{r.stderr}\n{r.stdout}")


def _compile_nodes():
    """Host code against PyTorch's and Python's headers."""
    import sysconfig

    import torch

    root = os.path.join(os.path.dirname(torch.__file__), "include")
    cuda = os.path.join(os.path.dirname(os.path.dirname(os.path.realpath(nvcc_path()))), "include")
    include = [SRC, root, os.path.join(root, "torch", "csrc", "api", "include"), cuda, sysconfig.get_paths()["include"]]
    obj = os.path.join(OBJ_DIR, NODES_SRC + ".o")
    _run(["g++", "-O2", "-std=c++17", "-fPIC", "-fvisibility=hidden", "-DTORCH_EXTENSION_NAME=_choco_autograd",
          f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}"] + [f"-I{d}" for d in include]
         + ["-c", os.path.join(SRC, NODES_SRC), "-o", obj], f"compiling {NODES_SRC}")
    return obj


def _link_nodes(obj):
    import torch

    libs = os.path.join(os.path.dirname(torch.__file__), "lib")
    _run(["g++", "-shared", "-o", NODES, obj, f"-L{OUT_DIR}", "-l:" + os.path.basename(LIB), f"-L{libs}", "-lc10", "-lc10_cuda", "-ltorch_cpu",
          "-ltorch_python", "-Wl,-rpath,$ORIGIN"], f"linking {os.path.basename(NODES)}")


def build(force=False, verbose=False):
    """Compile every source for sm_100a and link the shared library.  Returns its path."""
    if not force and is_current():
        return LIB
    nvcc = nvcc_path()
    if nvcc is None:
        if os.path.exists(LIB) and os.path.exists(NODES):
            return LIB
        raise RuntimeError("nvcc not found and no prebuilt library present")
    os.makedirs(OBJ_DIR, exist_ok=True)
    cu, cpp = sources()
    log = {}

    def compile_one(f):
        obj = os.path.join(OBJ_DIR, f + ".o")
        if f.endswith(".cu"):
            cmd = [nvcc] + NVCC_FLAGS + ["-I", SRC, "-c", os.path.join(SRC, f), "-o", obj]
        else:
            cmd = [nvcc, "-x", "c++", "-std=c++17", "-O3", "-Xcompiler", "-fPIC,-fopenmp", "-I", SRC, "-c",
                   os.path.join(SRC, f), "-o", obj]
        r = subprocess.run(cmd, capture_output=True, text=True)
        log[f] = r.stderr + r.stdout
        if r.returncode != 0:
            raise RuntimeError(f"compiling {f} failed:\n{r.stderr}\n{r.stdout}")
        return obj

    with ThreadPoolExecutor(max_workers=min(8, os.cpu_count() or 1)) as ex:
        nodes = ex.submit(_compile_nodes)          # the longest compilation starts first
        objs = list(ex.map(compile_one, cu + cpp))
        nodes_obj = nodes.result()
    link = [nvcc, "-shared", "-o", LIB] + objs + ["-Xcompiler", "-fopenmp", "-lgomp"]
    r = subprocess.run(link, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError("link failed:\n" + r.stderr + r.stdout)
    _link_nodes(nodes_obj)
    with open(os.path.join(OUT_DIR, "build.stamp"), "w") as fh:
        fh.write(_digest())
    with open(os.path.join(OUT_DIR, "ptxas.log"), "w") as fh:
        for f in cu:
            fh.write(f"==== {f}\n{log.get(f, '')}\n")
    if verbose:
        print(open(os.path.join(OUT_DIR, "ptxas.log")).read())
    return LIB


if __name__ == "__main__":
    path = build(force="--force" in sys.argv, verbose="--verbose" in sys.argv)
    print(path)
