"""Build the sm_100a shared library ``iris_kernel/libiris_b200.so`` and the
Python bindings ``iris_kernel/_ops.so`` in-tree.

    python iris-kernel_b200/build.py [--force]

Plain nvcc: the library exposes only the C ABI declared in
``include/iris_b200.h``.  The bindings are one C++ file over that ABI and
torch's headers, which calls what ctypes would, without a Python layer's time.  IEEE
division / square root stay on (no ``--use_fast_math``): the write path must
be bit-exact.  The library knows nothing of torch; the bindings are built anew
where torch or Python is another one than they were built for.
"""
from __future__ import annotations

import importlib.util
import os
import shutil
import subprocess
import sys
import sysconfig

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
CSRC = os.path.join(HERE, "csrc")
INCLUDE = os.path.join(ROOT, "include")
OUT = os.path.join(HERE, "iris_kernel", "libiris_b200.so")
BINDINGS = os.path.join(HERE, "iris_kernel", "_ops.so")
SOURCES = ["append.cu", "mrope_append.cu", "gather.cu", "decode.cu", "decode_noalloc.cu", "page_index.cu",
           "sparse_decode.cu", "varlen_attention.cu", "attention_mass.cu", "evict.cu", "exchange.cu"]

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-O3", "-lineinfo", "-std=c++17",
    "-Xcompiler", "-fPIC,-O2,-fvisibility=hidden",
    "-Xptxas", "-warn-spills",
    "--shared",
]


def _stamp():
    spec = importlib.util.spec_from_file_location("iris_ops_stamp", os.path.join(HERE, "iris_kernel", "_stamp.py"))
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def _nvcc() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found")


def _stale() -> bool:
    if not os.path.exists(OUT) or _bindings_stale():
        return True
    t = min(os.path.getmtime(OUT), os.path.getmtime(BINDINGS))
    deps = [os.path.join(CSRC, f) for f in os.listdir(CSRC)] + [os.path.join(INCLUDE, "iris_b200.h"), __file__]
    return any(os.path.getmtime(d) > t for d in deps)


def _bindings_stale() -> bool:
    stamp = _stamp()
    return not os.path.exists(BINDINGS) or stamp.built() != stamp.present()


def _run(cmd: list, verbose: bool) -> None:
    if verbose:
        print(" ".join(cmd))
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"{cmd[0]} failed ({res.returncode}):\n{res.stdout}\n{res.stderr}")
    if verbose and (res.stdout or res.stderr):
        print(res.stdout, res.stderr)


def _bindings_command() -> list:
    import torch

    root = os.path.dirname(torch.__file__)
    cuda = os.path.dirname(os.path.dirname(os.path.realpath(_nvcc())))
    include = [os.path.join(root, "include"), os.path.join(root, "include", "torch", "csrc", "api", "include"),
               os.path.join(cuda, "include"), sysconfig.get_paths()["include"]]
    return [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-shared", "-fPIC", "-fvisibility=hidden",
            f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", "-I", INCLUDE,
            *[x for d in include for x in ("-isystem", d)], os.path.join(CSRC, "bindings.cpp"),
            "-o", BINDINGS + ".tmp", "-L", os.path.dirname(OUT), "-l:libiris_b200.so", "-L", os.path.join(root, "lib"),
            "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch_cuda", "-ltorch_python", "-Wl,-rpath,$ORIGIN"]


def build(force: bool = False, verbose: bool = False) -> str:
    if not force and not _stale():
        return OUT
    cmd = [_nvcc(), "--threads", "0", *NVCC_FLAGS, "-I", INCLUDE, "-o", OUT + ".tmp", *[os.path.join(CSRC, s) for s in SOURCES]]
    _run(cmd, verbose)
    os.replace(OUT + ".tmp", OUT)
    _run(_bindings_command(), verbose)
    stamp = _stamp()
    if os.path.exists(stamp.PATH):
        os.remove(stamp.PATH)
    os.replace(BINDINGS + ".tmp", BINDINGS)
    with open(stamp.PATH, "w") as f:
        f.write(stamp.present() + "\n")
    return OUT


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose=True))
