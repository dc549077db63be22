"""Builds libfeather_b200.so (the C-ABI library declared in include/feather_b200.h) in-tree with nvcc for sm_100a, and
the torch binding of the MXFP4 operators and the fused norm (csrc/binding.cpp) with the C++ compiler.  The binding's file name carries
the Python and the torch it is for; where its tools are missing (``binding_unavailable()``) only the library is built.

Usage: ``python build.py`` from any directory, or ``build_all()``, ``build_library()`` and ``build_binding()`` from Python.  nvcc cross-compiles, so no GPU is
needed to build.  The library links the CUDA runtime statically and resolves the one driver symbol it needs
(cuTensorMapEncodeTiled) at run time, so it also loads on a machine without a driver (every call then reports an error).
"""

import importlib.machinery
import os
import shutil
import subprocess
import sys
import sysconfig

PKG_DIR = os.path.dirname(os.path.abspath(__file__))
CSRC_DIR = os.path.join(PKG_DIR, "csrc")
LIB_PATH = os.path.join(PKG_DIR, "libfeather_b200.so")
SOURCES = ["scaled_mm.cu", "scaled_mm_ext.cu", "quant.cu", "small_m.cu", "exchange.cu", "mxfp4.cu", "mxfp4_mm.cu", "norm.cu"]
HEADERS = ["ptx.cuh", "mxfp4.cuh", "host_util.h", os.path.join("..", "..", "include", "feather_b200.h")]

NVCC_FLAGS = [
    "-gencode",
    "arch=compute_100a,code=sm_100a",
    "-lineinfo",
    "-O3",
    "-std=c++17",
    "--cudart",
    "static",
    "-Xcompiler",
    "-fPIC",
    "-Xcompiler",
    "-fvisibility=hidden",
]


def _nvcc():
    nvcc = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(nvcc):
        raise RuntimeError("nvcc not found: libfeather_b200.so cannot be built")
    return nvcc


def is_stale():
    if not os.path.exists(LIB_PATH):
        return True
    built = os.path.getmtime(LIB_PATH)
    deps = [os.path.join(CSRC_DIR, s) for s in SOURCES + HEADERS]
    return any(os.path.getmtime(d) > built for d in deps if os.path.exists(d))


def build_library(force=False, verbose=False):
    """Compile every .cu under csrc/ into libfeather_b200.so.  Returns the library path."""
    if not force and not is_stale():
        return LIB_PATH
    nvcc = _nvcc()
    objs = []
    build_dir = os.path.join(PKG_DIR, "build")
    os.makedirs(build_dir, exist_ok=True)
    procs = []
    for src in SOURCES:
        obj = os.path.join(build_dir, src.replace(".cu", ".o"))
        cmd = [nvcc, *NVCC_FLAGS, "-c", os.path.join(CSRC_DIR, src), "-o", obj]
        if verbose:
            cmd.insert(1, "-Xptxas")
            cmd.insert(2, "-v")
        procs.append((src, subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)))
        objs.append(obj)
    for src, proc in procs:
        out, _ = proc.communicate()
        if verbose and out:
            print(out)
        if proc.returncode != 0:
            raise RuntimeError(f"nvcc failed on {src}:\n{out}")
    tmp = LIB_PATH + ".tmp"
    link = [nvcc, "-shared", "--cudart", "static", "-Xcompiler", "-fPIC", "-o", tmp, *objs]
    res = subprocess.run(link, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"link failed:\n{res.stdout}")
    os.replace(tmp, LIB_PATH)
    return LIB_PATH


BINDING_SRC = os.path.join(CSRC_DIR, "binding.cpp")


def binding_path():
    """Where the binding for this Python and this torch lies (the loader, kernel/b200/native.py, means the same file)."""
    import torch

    return os.path.join(PKG_DIR, f"_feather_binding.torch-{torch.__version__}{importlib.machinery.EXTENSION_SUFFIXES[0]}")


def _cxx():
    return shutil.which("c++") or shutil.which("g++")


def binding_unavailable():
    """What this machine lacks to build the binding, or None.  The library and the fp8 linear need none of it."""
    try:
        import torch
    except ImportError:
        return "torch is not installed"
    if _cxx() is None:
        return "there is no C++ compiler"
    if not os.path.exists(os.path.join(sysconfig.get_paths()["include"], "Python.h")):
        return "the headers of Python are not installed"
    if not os.path.exists(os.path.join(os.path.dirname(torch.__file__), "include", "ATen", "core", "Tensor.h")):
        return "the headers of torch are not installed"
    return None


def build_binding(force=False):
    """Compile csrc/binding.cpp against the installed torch.  Returns the path.  The module takes the entry points of
    libfeather_b200.so as addresses when it is loaded, so the two are built independently."""
    import torch

    path, cxx = binding_path(), _cxx()
    deps = [BINDING_SRC, os.path.join(PKG_DIR, "..", "include", "feather_b200.h"), torch.__file__]
    if not force and os.path.exists(path) and all(os.path.getmtime(d) <= os.path.getmtime(path) for d in deps):
        return path
    reason = binding_unavailable()
    if reason is not None:
        raise RuntimeError(f"the torch binding cannot be built: {reason}")
    torch_dir = os.path.dirname(torch.__file__)
    include = os.path.join(torch_dir, "include")
    cuda = os.path.dirname(os.path.dirname(_nvcc()))
    tmp = path + ".tmp"
    cmd = [cxx, "-O2", "-std=c++17", "-fPIC", "-shared", "-Wall", "-fvisibility=hidden", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
           "-I", include, "-I", os.path.join(include, "torch", "csrc", "api", "include"), "-I", sysconfig.get_paths()["include"], "-I", os.path.join(cuda, "include"),
           BINDING_SRC, "-L", os.path.join(torch_dir, "lib"), "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch_cuda", "-ltorch", "-ltorch_python", "-o", tmp]
    res = subprocess.run(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"torch binding failed to build:\n{res.stdout}")
    os.replace(tmp, path)
    return path


def build_all(force=False, verbose=False):
    """The library and, where its tools are there, the binding.  Returns their paths."""
    paths = [build_library(force=force, verbose=verbose)]
    reason = binding_unavailable()
    if reason is None:
        paths.append(build_binding(force=force))
    else:
        print(f"torch binding not built: {reason} (the MXFP4 operators and the fused norm will not be available)", file=sys.stderr)
    return paths


CBENCH_SRC = os.path.join(PKG_DIR, "cbench", "bench_scaled_mm.c")
CBENCH_BIN = os.path.join(PKG_DIR, "cbench", "bench_scaled_mm")


def build_cbench(cc=None):
    """Compile cbench/bench_scaled_mm.c - plain C against include/feather_b200.h, linked with the library and the CUDA runtime."""
    build_library()
    cc = cc or shutil.which("cc") or shutil.which("gcc")
    if cc is None:
        raise RuntimeError("no C compiler found")
    cuda = os.path.dirname(os.path.dirname(_nvcc()))
    cmd = [cc, "-std=c99", "-O2", "-Wall", "-Wextra", "-pedantic", CBENCH_SRC, "-I", os.path.join(PKG_DIR, "..", "include"), "-I", os.path.join(cuda, "include"),
           "-L", PKG_DIR, "-lfeather_b200", "-L", os.path.join(cuda, "lib64"), "-lcudart", "-lm", "-Wl,-rpath," + PKG_DIR,
           "-Wl,-rpath," + os.path.join(cuda, "lib64"), "-o", CBENCH_BIN]
    res = subprocess.run(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"C harness failed to build:\n{res.stdout}")
    return CBENCH_BIN


if __name__ == "__main__":
    for path in build_all(force="--force" in sys.argv, verbose="-v" in sys.argv):
        print(path)
    if "--cbench" in sys.argv:
        print(build_cbench())
