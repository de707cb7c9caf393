"""In-tree build of libflexkv_b200.so (sm_100a) with nvcc.

    python -m flexkv_b200.build          # build if sources are newer
    python -m flexkv_b200.build --force  # always rebuild

The library lands in flexkv_b200/_lib/ so it travels with the source tree;
no JIT cache is involved.  `-Xptxas -v` output (registers, spills, shared
memory per kernel) is written next to it as ptxas.txt.
"""
from __future__ import annotations

import argparse
import importlib.metadata
import os
import shutil
import subprocess
import sys
import sysconfig
import warnings

PKG_DIR = os.path.dirname(os.path.abspath(__file__))
REPO_DIR = os.path.dirname(PKG_DIR)
CSRC = os.path.join(PKG_DIR, "csrc")
LIB_DIR = os.path.join(PKG_DIR, "_lib")
LIB_PATH = os.path.join(LIB_DIR, "libflexkv_b200.so")
BINDING = os.path.join(CSRC, "fp4_binding.cpp")  # the 4-bit cache's operators on torch tensors
BINDING_HEADERS = [os.path.join(CSRC, "fp4_overlap.h"), os.path.join(REPO_DIR, "include", "flexkv_b200.h")]
SOURCES = ["fkv_common.cpp", "transfer.cu", "tp_group.cpp", "xxh64.cu", "engine.cpp", "ipc.cpp", "ssd.cpp",
           "block_index.cu", "fp4_cache.cu", "fp4_attention.cu"]
HEADERS = [os.path.join(CSRC, "fkv_common.h"), os.path.join(CSRC, "fp4_format.cuh"), os.path.join(CSRC, "fp4_launch.cuh"),
           os.path.join(CSRC, "fp4_wait.cuh"),
           os.path.join(REPO_DIR, "include", "flexkv_b200.h")]
ARCH_FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a"]


def _nvcc() -> str:
    for cand in (os.environ.get("NVCC"), "/usr/local/cuda/bin/nvcc", shutil.which("nvcc")):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found; set NVCC or install the CUDA toolkit")


def _stale() -> bool:
    if not os.path.exists(LIB_PATH):
        return True
    t = os.path.getmtime(LIB_PATH)
    deps = [os.path.join(CSRC, s) for s in SOURCES] + HEADERS + [os.path.abspath(__file__)]
    return any(os.path.getmtime(d) > t for d in deps)


def binding_path() -> str:
    """Where the 4-bit cache's CPython module is for this interpreter and this
    torch: its layouts of tensors and exceptions are those of the headers it
    was built with, so another version gets a module of its own."""
    if "torch" in sys.modules:
        torch = sys.modules["torch"].__version__
    else:  # a build with nothing to do need not import it
        try:
            torch = importlib.metadata.version("torch")
        except importlib.metadata.PackageNotFoundError:
            torch = "none"
    return os.path.join(LIB_DIR, f"_fp4.{sysconfig.get_config_var('SOABI')}.torch-{torch}.so")


def _binding_includes() -> list:
    import torch.utils.cpp_extension

    return [sysconfig.get_paths()["include"], *torch.utils.cpp_extension.include_paths()]


def _binding_lacks() -> str:
    """What the module cannot be built without and is not there; the library
    needs neither."""
    try:
        inc = _binding_includes()
    except ImportError as e:
        return str(e)
    for header in ("Python.h", os.path.join("torch", "csrc", "autograd", "python_variable.h")):
        if not any(os.path.exists(os.path.join(d, header)) for d in inc):
            return f"{header} not found"
    return ""


def _build_binding(verbose: bool) -> None:
    """The CPython module of the 4-bit cache's operators, against this
    interpreter and the installed torch."""
    import torch

    torch_lib = os.path.join(os.path.dirname(torch.__file__), "lib")
    inc = _binding_includes()
    tmp = binding_path() + ".tmp"
    # The C++ library has to be the shared one that torch uses: a second copy, linked statically as some
    # compilers' defaults have it, ends the process at the first stream or exception that meets the other.
    cmd = [
        _nvcc(), "-O2", "-std=c++17", "-Xcompiler", "-fPIC,-Wall", "-shared",
        f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
        *[a for d in inc for a in ("-isystem", d)], "-o", tmp, BINDING, f"-L{torch_lib}", "-ltorch_python", "-ltorch",
        "-ltorch_cpu", "-lc10", "-lc10_cuda", "-Xlinker", f"-rpath={torch_lib}", "-Xlinker", "-l:libstdc++.so.6",
        "-cudart", "none",
    ]
    if verbose:
        print(" ".join(cmd))
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"{cmd[0]} failed ({res.returncode}):\n{res.stderr[-4000:]}")
    os.replace(tmp, binding_path())


def _binding_stale() -> bool:
    path = binding_path()
    if not os.path.exists(path):
        return True
    deps = [BINDING, *BINDING_HEADERS, os.path.abspath(__file__)]
    return any(os.path.getmtime(d) > os.path.getmtime(path) for d in deps)


def build(force: bool = False, verbose: bool = False) -> str:
    """Builds what is out of date; returns the library's path.  Without the
    headers of Python or torch the library alone is built, with a warning:
    ``fp4_cache`` then raises ImportError when it is used."""
    lib = _build_lib(force, verbose)
    if force or _binding_stale():
        lacks = _binding_lacks()
        if lacks:
            warnings.warn(f"flexkv_b200.fp4_cache is not built: {lacks}")
        else:
            _build_binding(verbose)
    return lib


def _build_lib(force: bool, verbose: bool) -> str:
    if not force and not _stale():
        return LIB_PATH
    os.makedirs(LIB_DIR, exist_ok=True)
    tmp = LIB_PATH + ".tmp"
    cmd = [
        _nvcc(), *ARCH_FLAGS, "-O3", "-lineinfo", "-std=c++17",
        "-Xcompiler", "-fPIC,-O3,-Wall", "-Xptxas", "-v", "--threads", "0", "-shared",
        "-I", os.path.join(REPO_DIR, "include"),
        "-o", tmp, *[os.path.join(CSRC, s) for s in SOURCES], "-lpthread",
    ]
    if verbose:
        print(" ".join(cmd))
    res = subprocess.run(cmd, capture_output=True, text=True)
    with open(os.path.join(LIB_DIR, "ptxas.txt"), "w") as f:
        f.write(res.stdout)
        f.write(res.stderr)
    if res.returncode != 0:
        raise RuntimeError(f"nvcc failed ({res.returncode}):\n{res.stderr[-4000:]}")
    os.replace(tmp, LIB_PATH)
    return LIB_PATH


def main(argv=None) -> int:
    ap = argparse.ArgumentParser()
    ap.add_argument("--force", action="store_true")
    ap.add_argument("-v", "--verbose", action="store_true")
    a = ap.parse_args(argv)
    print(build(force=a.force, verbose=a.verbose))
    return 0


if __name__ == "__main__":
    sys.exit(main())
