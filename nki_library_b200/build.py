"""Build the CUDA shared library in-tree with nvcc for sm_100a, and the torch side of the training operators with g++.

``python -m nki_library_b200.build`` (or ``build_library()``) compiles every
``csrc/*.cu`` into ``nki_library_b200/libb200moe.so``, and ``csrc/autograd.cpp``
against it into ``nki_library_b200/_autograd.so``.  nvcc cross-compiles, so this
works on a machine without a GPU.
"""

from __future__ import annotations

import glob
import importlib.util
import os
import subprocess
import sys

PKG = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(PKG, "csrc")
LIB = os.path.join(PKG, "libb200moe.so")
AUTOGRAD = os.path.join(PKG, "_autograd.so")
BUILD = os.path.join(PKG, "build")

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a", "-lineinfo", "-O3", "-std=c++17",
    "-Xcompiler", "-fPIC", "--expt-relaxed-constexpr",
]


def _nvcc() -> str:
    cand = os.path.join(os.environ.get("CUDA_HOME", "/usr/local/cuda"), "bin", "nvcc")
    return cand if os.path.exists(cand) else "nvcc"


def _stale(target: str, deps) -> bool:
    if not os.path.exists(target):
        return True
    t = os.path.getmtime(target)
    return any(os.path.getmtime(d) > t for d in deps)


def _autograd_compile(source: str, target: str) -> list:
    import sysconfig

    import torch

    include = os.path.join(os.path.dirname(torch.__file__), "include")
    dirs = [include, os.path.join(include, "torch", "csrc", "api", "include"), sysconfig.get_paths()["include"],
            os.path.join(os.environ.get("CUDA_HOME", "/usr/local/cuda"), "include")]
    return (["g++", "-O2", "-std=c++17", "-fPIC", "-DTORCH_EXTENSION_NAME=_autograd",
             f"-D_GLIBCXX_USE_CXX11_ABI={int(torch.compiled_with_cxx11_abi())}"] +
            [a for d in dirs for a in ("-isystem", d)] + ["-c", source, "-o", target])


def _autograd_link(target: str) -> list:
    import torch

    return ["g++", "-shared", "-o", AUTOGRAD, target, "-L" + os.path.join(os.path.dirname(torch.__file__), "lib"),
            "-ltorch_python", "-ltorch", "-ltorch_cpu", "-lc10_cuda", "-lc10", "-L" + PKG, "-l:" + os.path.basename(LIB),
            "-Wl,-rpath,$ORIGIN"]


def _report(command: list, out: str, verbose: bool, failed: bool) -> None:
    if failed or verbose:
        sys.stderr.write(out or " ".join(command) + "\n")


def _write_stamp() -> bool:
    """Names the torch and the Python that the torch side is compiled against beside it; whether these are others than before."""
    import sysconfig

    import torch

    path = os.path.join(BUILD, "autograd.stamp")
    text = f"{torch.__version__} {os.path.dirname(torch.__file__)} {sysconfig.get_config_var('SOABI')}\n"
    if os.path.exists(path):
        with open(path) as f:
            if f.read() == text:
                return False
    with open(path, "w") as f:
        f.write(text)
    return True


def _start_autograd(hdr: str, force: bool):
    """The running compiler of the torch side, None if there is nothing to compile."""
    source, obj = os.path.join(CSRC, "autograd.cpp"), os.path.join(BUILD, "autograd.o")
    if _write_stamp() and os.path.exists(obj):
        os.remove(obj)
    if not (force or _stale(obj, [source, hdr])):
        return None
    return subprocess.Popen(_autograd_compile(source, obj), stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)


def _finish_autograd(compiler, force: bool, verbose: bool) -> None:
    obj = os.path.join(BUILD, "autograd.o")
    if compiler is not None:
        out, _ = compiler.communicate()
        _report(compiler.args, out, verbose, compiler.returncode != 0)
        if compiler.returncode != 0:
            raise RuntimeError("compilation failed")
    if force or _stale(AUTOGRAD, [obj]):
        subprocess.check_call(_autograd_link(obj))


def build_library(force: bool = False, verbose: bool = False) -> str:
    """The shared library; raises if it cannot be built.  The torch side is built beside it where torch is installed.  A C program
    needs neither, so what goes wrong there (no Python headers, a torch without CUDA) is reported and leaves the library as it is;
    the training operators then raise on their first call."""
    srcs = sorted(glob.glob(os.path.join(CSRC, "*.cu")))
    hdrs = sorted(glob.glob(os.path.join(CSRC, "*.cuh"))) + [os.path.join(os.path.dirname(PKG), "include", "b200moe.h")]
    os.makedirs(BUILD, exist_ok=True)
    objs = []
    procs = []
    for s in srcs:
        o = os.path.join(BUILD, os.path.basename(s)[:-3] + ".o")
        objs.append(o)
        if force or _stale(o, [s] + hdrs):
            cmd = [_nvcc()] + NVCC_FLAGS + (["-Xptxas", "-v"] if verbose else []) + ["-c", s, "-o", o]
            procs.append(subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True))
    torch_side, trouble = None, None
    if importlib.util.find_spec("torch") is not None:
        try:
            torch_side = _start_autograd(hdrs[-1], force)
        except Exception as error:
            trouble = error
    else:
        trouble = "torch is not installed"
    failed = False
    for p in procs:
        out, _ = p.communicate()
        _report(p.args, out, verbose, p.returncode != 0)
        failed |= p.returncode != 0
    if failed:
        if torch_side is not None:
            torch_side.communicate()
        raise RuntimeError("compilation failed")
    if force or procs or _stale(LIB, objs):
        subprocess.check_call([_nvcc(), "-shared", "-o", LIB] + objs + ["-lcudart"])
    try:
        if trouble is None:
            _finish_autograd(torch_side, force, verbose)
    except Exception as error:
        trouble = error
    if trouble is not None:
        if os.path.exists(AUTOGRAD):  # it would fit an earlier library
            os.remove(AUTOGRAD)
        sys.stderr.write(f"{LIB} is built; {AUTOGRAD}, which the training operators need, is not: {trouble}\n")
    return LIB


if __name__ == "__main__":
    print(build_library(force="--force" in sys.argv, verbose="-v" in sys.argv))
