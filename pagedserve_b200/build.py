"""Build libpagedserve_b200.so in-tree with nvcc for sm_100a, and _calls.so,
the Python module of csrc/calls.cpp that calls it, with the host compiler.

    python -m pagedserve_b200.build            # incremental
    python -m pagedserve_b200.build --force    # rebuild everything

Objects go to ``pagedserve_b200/_build/``; the shared library lands next to
this file so it travels with the source tree.
"""

from __future__ import annotations

import argparse
import concurrent.futures as cf
import os
import shutil
import subprocess
import sys

PKG = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(PKG)
CSRC = os.path.join(PKG, "csrc")
BUILD = os.path.join(PKG, "_build")
LIB = os.path.join(PKG, "libpagedserve_b200.so")
CALLS_SRC = os.path.join(CSRC, "calls.cpp")
CALLS = os.path.join(PKG, "_calls.so")
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
FLAGS = ["-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC,-O2", "--expt-relaxed-constexpr",
         "-I", os.path.join(ROOT, "include")]


def nvcc() -> str:
    for cand in (os.environ.get("NVCC"), "/usr/local/cuda/bin/nvcc", shutil.which("nvcc")):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found")


def _deps() -> list[str]:
    hdrs = [os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith((".cuh", ".h"))]
    return hdrs + [os.path.join(ROOT, "include", "pagedserve_b200.h")]


def _compile(src: str, force: bool, extra: list[str]) -> str:
    obj = os.path.join(BUILD, os.path.basename(src) + ".o")
    newest_dep = max([os.path.getmtime(src)] + [os.path.getmtime(d) for d in _deps()])
    if not force and os.path.exists(obj) and os.path.getmtime(obj) >= newest_dep:
        return obj
    cmd = [nvcc(), *ARCH, *FLAGS, *extra, "-c", src, "-o", obj]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"nvcc failed for {src}:\n{res.stdout}\n{res.stderr}")
    return obj


def calls_target() -> str:
    """The torch, interpreter and C++ ABI that _calls.so is compiled for: it uses their internals."""
    import sysconfig

    import torch
    return f"torch {torch.__version__}, {sysconfig.get_config_var('EXT_SUFFIX')}, abi {int(torch._C._GLIBCXX_USE_CXX11_ABI)}"


def _calls_command() -> list[str]:
    """The compiler's command, but for its output: csrc/calls.cpp against this interpreter, this torch and LIB."""
    import sysconfig

    import torch
    base = os.path.dirname(torch.__file__)
    include = os.path.join(base, "include")
    cuda = os.path.dirname(os.path.dirname(nvcc()))
    return [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden",
            f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", f'-DPSB_BUILT_FOR="{calls_target()}"',
            "-I", os.path.join(ROOT, "include"), "-isystem", include,
            "-isystem", os.path.join(include, "torch", "csrc", "api", "include"),
            "-isystem", sysconfig.get_paths()["include"], "-isystem", os.path.join(cuda, "include"),
            CALLS_SRC, "-L", os.path.join(base, "lib"), "-ltorch_python", "-ltorch_cuda",
            "-ltorch_cpu", "-ltorch", "-lc10_cuda", "-lc10", "-L", PKG, "-l:libpagedserve_b200.so",
            "-Wl,-rpath,$ORIGIN"]


def _build_calls(force: bool) -> None:
    """_calls.so, unless it is newer than its sources and made by the same command for the same target."""
    cmd = _calls_command()
    key, stamp = "\n".join(cmd), os.path.join(BUILD, "calls.key")
    newest = max(os.path.getmtime(p) for p in (CALLS_SRC, os.path.join(ROOT, "include", "pagedserve_b200.h")))
    if not force and os.path.exists(CALLS) and os.path.getmtime(CALLS) >= newest and os.path.exists(stamp):
        with open(stamp) as f:
            if f.read() == key:
                return
    tmp = f"{CALLS}.{os.getpid()}.tmp"  # builds at once do not write into each other's
    res = subprocess.run(cmd + ["-o", tmp], capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"building {CALLS_SRC} failed:\n{res.stdout}\n{res.stderr}")
    os.replace(tmp, CALLS)
    with open(f"{stamp}.{os.getpid()}.tmp", "w") as f:
        f.write(key)
    os.replace(f.name, stamp)


def build(force: bool = False, verbose: bool = False, extra: list[str] | None = None) -> str:
    os.makedirs(BUILD, exist_ok=True)
    extra = list(extra or [])
    srcs = sorted(os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith(".cu"))
    with cf.ThreadPoolExecutor(max_workers=min(8, len(srcs))) as ex:
        objs = list(ex.map(lambda s: _compile(s, force, extra), srcs))
    if force or not os.path.exists(LIB) or os.path.getmtime(LIB) < max(os.path.getmtime(o) for o in objs):
        tmp = LIB + ".tmp"
        cmd = [nvcc(), *ARCH, "-shared", "-o", tmp, *objs, "-lcudart_static", "-lrt", "-lpthread", "-ldl"]
        res = subprocess.run(cmd, capture_output=True, text=True)
        if res.returncode != 0:
            raise RuntimeError(f"link failed:\n{res.stdout}\n{res.stderr}")
        os.replace(tmp, LIB)
    _build_calls(force)
    if verbose:
        print(LIB)
    return LIB


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--force", action="store_true")
    a = ap.parse_args()
    build(force=a.force, verbose=True)
    sys.exit(0)
