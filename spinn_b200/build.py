"""Builds libspinn_cuda.so in-tree with nvcc for sm_100a, and the torch binding of its
decoder-serving operators (_torch_ops.so) with the host compiler.

Usage: ``python -m spinn_b200.build [--force] [--verbose]``.  Object files go to
``spinn_b200/_build/`` and the shared library to ``spinn_b200/libspinn_cuda.so``; both are
git-ignored but travel with the working tree.  A source is recompiled when it or any header
under ``csrc/`` or ``include/`` is newer than its object.
"""
from __future__ import annotations

import argparse
import importlib.util
import os
import shutil
import subprocess
import sys
import sysconfig
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
CSRC = os.path.join(HERE, "csrc")
BUILD = os.path.join(HERE, "_build")
LIB = os.path.join(HERE, "libspinn_cuda.so")
TORCH_OPS = os.path.join(HERE, "_torch_ops.so")
SOURCES = ["tmap.cpp", "tc_gemm.cu", "glue.cu", "runtime.cpp", "abi.cpp", "noalloc.cu", "winograd.cu", "tail.cu",
           "cache.cu", "attention.cu", "attention_fp16.cu", "attention_bf16.cu", "attention_fp32.cu",
           "linear.cu"]

ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
COMMON = ["-O3", "-std=c++17", "-lineinfo", "-Xcompiler", "-fPIC,-fvisibility=hidden",
          "-I" + os.path.join(ROOT, "include"), "-I" + CSRC]


def nvcc() -> str:
    for cand in (os.environ.get("NVCC"), "/usr/local/cuda/bin/nvcc", shutil.which("nvcc")):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found")


def host_compiler() -> list:
    # The image exports CC/CXX pointing at a wrapper; nvcc is given the system g++.
    for cand in ("/usr/bin/g++", shutil.which("g++")):
        if cand and os.path.exists(cand):
            return ["-ccbin", cand]
    return []


def _headers_mtime() -> float:
    t = 0.0
    for d in (CSRC, os.path.join(ROOT, "include")):
        for f in os.listdir(d):
            if f.endswith((".h", ".cuh", ".hpp")):
                t = max(t, os.path.getmtime(os.path.join(d, f)))
    return t


def _compile(src: str, force: bool, verbose: bool, extra: list) -> str:
    obj = os.path.join(BUILD, os.path.splitext(src)[0] + ".o")
    path = os.path.join(CSRC, src)
    if not force and os.path.exists(obj):
        if os.path.getmtime(obj) >= max(os.path.getmtime(path), _headers_mtime()):
            return obj
    lang = ["-x", "cu"] if src.endswith(".cu") else ["-x", "c++"]
    cmd = [nvcc()] + host_compiler() + ARCH + COMMON + extra + lang + ["-c", path, "-o", obj]
    if verbose:
        print(" ".join(cmd), flush=True)
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"nvcc failed on {src}:\n{r.stdout}\n{r.stderr}")
    if verbose and (r.stdout.strip() or r.stderr.strip()):
        print(r.stdout + r.stderr, flush=True)
    return obj


def _build_torch_ops(force: bool, verbose: bool) -> None:
    """csrc/torch_ops.cpp against the installed torch; rebuilt when it, the C header or torch's
    version changes.  Without torch there is nothing to bind: the C library is complete by itself."""
    import importlib.metadata
    spec = importlib.util.find_spec("torch")
    if spec is None:
        print("spinn_b200: torch is not installed, its binding (_torch_ops.so) is not built", file=sys.stderr)
        return
    src = os.path.join(CSRC, "torch_ops.cpp")
    stamp = os.path.join(BUILD, "torch_ops.version")
    version = importlib.metadata.version("torch")
    newest = max(os.path.getmtime(src), _headers_mtime())
    if not force and os.path.exists(TORCH_OPS) and os.path.exists(stamp) and \
            os.path.getmtime(TORCH_OPS) >= newest and open(stamp).read() == version:
        return
    root = os.path.dirname(spec.origin)
    cxx = host_compiler()[-1] if host_compiler() else "g++"
    cmd = [cxx, "-O2", "-std=c++20", "-fPIC", "-shared", "-fvisibility=hidden", "-I" + os.path.join(root, "include"),
           "-I" + os.path.join(root, "include", "torch", "csrc", "api", "include"),
           "-I" + os.path.join(os.path.dirname(os.path.dirname(nvcc())), "include"),
           "-I" + sysconfig.get_paths()["include"], src, "-o", TORCH_OPS, "-L" + HERE, "-l:libspinn_cuda.so",
           "-L" + os.path.join(root, "lib"), "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch_python",
           "-Wl,-rpath,$ORIGIN"]
    if verbose:
        print(" ".join(cmd), flush=True)
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"{cxx} failed on torch_ops.cpp:\n{r.stdout}\n{r.stderr}")
    with open(stamp, "w") as f:
        f.write(version)


def build(force: bool = False, verbose: bool = False, ptxas_verbose: bool = False) -> str:
    os.makedirs(BUILD, exist_ok=True)
    extra = ["-Xptxas", "-v"] if ptxas_verbose else []
    with ThreadPoolExecutor(max_workers=len(SOURCES)) as ex:
        objs = list(ex.map(lambda s: _compile(s, force, verbose or ptxas_verbose, extra), SOURCES))
    newest = max(os.path.getmtime(o) for o in objs)
    if force or not os.path.exists(LIB) or os.path.getmtime(LIB) < newest:
        cmd = [nvcc()] + host_compiler() + ARCH + ["-shared", "-o", LIB] + objs + ["-lpthread"]
        if verbose:
            print(" ".join(cmd), flush=True)
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"link failed:\n{r.stdout}\n{r.stderr}")
    _build_torch_ops(force, verbose)
    return LIB


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--force", action="store_true")
    ap.add_argument("--verbose", action="store_true")
    ap.add_argument("--ptxas-verbose", action="store_true")
    a = ap.parse_args()
    print(build(a.force, a.verbose, a.ptxas_verbose))
    sys.exit(0)
