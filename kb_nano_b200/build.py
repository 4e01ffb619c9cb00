"""Builds libkbn_fp8.so (the C-ABI CUDA library) in-tree with nvcc for sm_100a, and _calls.so (the native call path of the
small operators, csrc/calls.cpp, which reads torch tensors itself) with g++.

    python -m kb_nano_b200.build [--force] [--verbose]

Either is rebuilt only when a source or header is newer than it, _calls.so also when torch, Python or its compiler flags are not
the ones it was built with (build/_calls.stamp).  Each is linked beside its place and moved there whole, so that a process that
loads it during a build finds the old or the new one.  nvcc cross-compiles without a GPU, so this also serves as the "does it
build" check on a CPU-only machine.
"""
from __future__ import annotations

import concurrent.futures
import glob
import os
import shutil
import subprocess
import sys

PKG_DIR = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(PKG_DIR, "csrc")
INCLUDE = os.path.join(os.path.dirname(PKG_DIR), "include")
LIB_PATH = os.path.join(PKG_DIR, "libkbn_fp8.so")
OBJ_DIR = os.path.join(PKG_DIR, "build")
CALLS_SRC = os.path.join(CSRC, "calls.cpp")
CALLS_PATH = os.path.join(PKG_DIR, "_calls.so")
CALLS_STAMP = os.path.join(OBJ_DIR, "_calls.stamp")
CALLS_FLAGS = ["-O2", "-std=c++17", "-shared", "-fPIC", "-fvisibility=hidden"]

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-O3", "-std=c++17", "-lineinfo",
    "-Xcompiler", "-fPIC",
    "-Xptxas", "-v",
]


def _nvcc() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found: set $NVCC or put nvcc on PATH")


def sources() -> list[str]:
    return sorted(glob.glob(os.path.join(CSRC, "*.cu")))


def _deps() -> list[str]:
    return sources() + glob.glob(os.path.join(CSRC, "*.cuh")) + glob.glob(os.path.join(INCLUDE, "*.h"))


def needs_build() -> bool:
    if not os.path.exists(LIB_PATH):
        return True
    t = os.path.getmtime(LIB_PATH)
    return any(os.path.getmtime(f) > t for f in _deps())


def _compile_one(nvcc: str, src: str, verbose: bool) -> tuple[str, str]:
    obj = os.path.join(OBJ_DIR, os.path.basename(src)[:-3] + ".o")
    cmd = [nvcc, *NVCC_FLAGS, "-I", INCLUDE, "-c", src, "-o", obj]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"nvcc failed on {src}:\n{r.stdout}\n{r.stderr}")
    return obj, r.stderr if verbose else ""


def _link(cmd: list[str], path: str, what: str) -> None:
    """Runs `cmd` + -o with a file beside `path`, then moves that file there."""
    tmp = f"{path}.{os.getpid()}.tmp"
    try:
        r = subprocess.run([*cmd, "-o", tmp], capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"{what} failed:\n{r.stdout}\n{r.stderr}")
        os.replace(tmp, path)
    finally:
        if os.path.exists(tmp):
            os.remove(tmp)


def _calls_command() -> list[str]:
    import sysconfig

    import torch
    root = os.path.dirname(torch.__file__)
    cuda = os.path.dirname(os.path.dirname(os.path.realpath(_nvcc())))
    include = [INCLUDE, os.path.join(root, "include"), os.path.join(root, "include", "torch", "csrc", "api", "include"),
               os.path.join(cuda, "include"), sysconfig.get_paths()["include"]]
    lib = os.path.join(root, "lib")
    return [shutil.which("g++") or "g++", *CALLS_FLAGS,
            f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", *(f"-I{d}" for d in include), CALLS_SRC,
            f"-L{PKG_DIR}", "-l:" + os.path.basename(LIB_PATH), f"-L{lib}", "-ltorch_python", "-ltorch_cpu", "-lc10", "-lc10_cuda",
            "-Wl,-rpath,$ORIGIN", f"-Wl,-rpath,{lib}"]


def _calls_stamp() -> str:
    """What _calls.so depends on beside its sources (torch and Python promise no binary layout), known without a compiler at hand."""
    import torch
    return "\n".join([torch.__version__, torch.__file__, str(torch._C._GLIBCXX_USE_CXX11_ABI), sys.version, *CALLS_FLAGS])


def _calls_need_build() -> bool:
    if not os.path.exists(CALLS_PATH) or not os.path.exists(CALLS_STAMP):
        return True
    t = os.path.getmtime(CALLS_PATH)
    if any(os.path.getmtime(f) > t for f in (CALLS_SRC, os.path.join(INCLUDE, "kbn_fp8.h"))):
        return True
    with open(CALLS_STAMP) as f:
        return f.read() != _calls_stamp()


def _build_calls() -> None:
    os.makedirs(os.path.dirname(CALLS_STAMP), exist_ok=True)
    if os.path.exists(CALLS_STAMP):
        os.remove(CALLS_STAMP)           # an interrupted build is not taken for a finished one
    _link(_calls_command(), CALLS_PATH, f"g++ on {CALLS_SRC}")
    with open(CALLS_STAMP, "w") as f:
        f.write(_calls_stamp())


def build(force: bool = False, verbose: bool = False) -> str:
    _build_lib(force, verbose)
    if force or _calls_need_build():
        _build_calls()
    return LIB_PATH


def _build_lib(force: bool, verbose: bool) -> str:
    if not force and not needs_build():
        return LIB_PATH
    nvcc = _nvcc()
    os.makedirs(OBJ_DIR, exist_ok=True)
    srcs = sources()
    with concurrent.futures.ThreadPoolExecutor(max_workers=min(8, len(srcs))) as ex:
        results = list(ex.map(lambda s: _compile_one(nvcc, s, verbose), srcs))
    objs = [o for o, _ in results]
    if verbose:
        for _, log in results:
            sys.stderr.write(log)
    _link([nvcc, "-shared", *objs, "-cudart", "static", "-Xcompiler", "-fPIC"], LIB_PATH, "linking the library")
    return LIB_PATH


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="--verbose" in sys.argv))
