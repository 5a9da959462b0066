"""Builds ``libarboretum.so`` in-tree with nvcc for sm_100a.

    python arboretum_b200/build.py [--force]

The library is the product: the C ABI the Python layer (and the reference's own
``core.py``) loads with ctypes.  nvcc cross-compiles without a GPU.
"""
import os
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
BUILD = os.path.join(HERE, "_build")
LIB = os.path.join(HERE, "libarboretum.so")
SOURCES = ["abi.cu", "garden.cu", "hist.cu", "split.cu", "partition.cu", "objective.cu", "quantize.cu", "exchange.cu",
           "lookup.cu", "adamw.cu", "operators_abi.cu"]
HEADERS = ["common.cuh", "config.h", "gain.cuh", "garden.h", "json.h", "kernels.cuh", "exchange.h", "abi.h", "operators.h",
           "vec.cuh", "root.cuh"]
BINDINGS = os.path.join(HERE, "_tensors.so")  # the operators on torch tensors
NVCC = os.environ.get("NVCC", "nvcc")
FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a", "-lineinfo", "-O3", "-std=c++17",
         "--fmad=false", "-Xcompiler", "-fPIC", "-Xptxas", "-v", "-ccbin", "/usr/bin/g++"]


def _stale(target, deps):
    if not os.path.exists(target):
        return True
    t = os.path.getmtime(target)
    return any(os.path.getmtime(d) > t for d in deps)


def _compile(src):
    obj = os.path.join(BUILD, src.replace(".cu", ".o"))
    deps = [os.path.join(CSRC, src)] + [os.path.join(CSRC, h) for h in HEADERS] + \
           [os.path.join(HERE, "..", "include", "arboretum_b200.h")]
    if not _stale(obj, deps):
        return obj, ""
    cmd = [NVCC] + FLAGS + ["-c", os.path.join(CSRC, src), "-o", obj]
    r = subprocess.run(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)
    if r.returncode != 0:
        raise RuntimeError("nvcc failed for %s:\n%s" % (src, r.stdout))
    with open(obj + ".log", "w") as f:
        f.write(r.stdout)
    return obj, r.stdout


def _bindings():
    """The Python module of the operators on torch tensors: g++ against torch's headers, linked to
    the library beside it."""
    import sysconfig
    try:
        import torch
        from torch.utils import cpp_extension
    except ImportError as e:
        print("the operators on torch tensors are left out: %s" % e)
        return
    src = os.path.join(CSRC, "bindings.cpp")
    if not _stale(BINDINGS, [src, os.path.join(HERE, "..", "include", "arboretum_b200.h")]):
        return
    include = cpp_extension.include_paths() + [sysconfig.get_paths()["include"], "/usr/local/cuda/include"]
    lib = os.path.join(os.path.dirname(torch.__file__), "lib")
    cmd = ["/usr/bin/g++", "-O2", "-std=c++17", "-shared", "-fPIC",
           "-D_GLIBCXX_USE_CXX11_ABI=%d" % int(torch._C._GLIBCXX_USE_CXX11_ABI)]
    cmd += [x for d in include for x in ("-isystem", d)]
    cmd += [src, "-o", BINDINGS, "-L" + HERE, "-l:libarboretum.so", "-Wl,-rpath,$ORIGIN", "-L" + lib,
            "-ltorch_python", "-ltorch", "-ltorch_cpu", "-lc10", "-lc10_cuda"]
    r = subprocess.run(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)
    if r.returncode != 0:
        raise RuntimeError("g++ failed for bindings.cpp:\n" + r.stdout)


def build(force=False, verbose=False):
    os.makedirs(BUILD, exist_ok=True)
    if force:
        for f in os.listdir(BUILD):
            os.remove(os.path.join(BUILD, f))
    with ThreadPoolExecutor(max_workers=min(8, len(SOURCES))) as ex:
        results = list(ex.map(_compile, SOURCES))
    objs = [o for o, _ in results]
    if verbose:
        for _, log in results:
            if log:
                print(log)
    if _stale(LIB, objs):
        cmd = [NVCC, "-shared", "-o", LIB] + objs + ["-ldl", "-ccbin", "/usr/bin/g++"]
        r = subprocess.run(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)
        if r.returncode != 0:
            raise RuntimeError("link failed:\n" + r.stdout)
    _bindings()
    return LIB


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose=True))
