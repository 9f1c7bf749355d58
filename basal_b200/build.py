"""Builds libbasal200.so (every CUDA kernel of the package, sm_100a only) and libbasal200_torch-<torch version>.so (the torch
ops that are registered in C++, which call it) next to this file.

    python basal_b200/build.py [--force]    (a plain script: importing basal_b200 needs libbasal200.so)

nvcc cross-compiles without a GPU. libbasal200.so links the CUDA runtime statically and resolves the one driver
function it needs (cuTensorMapEncodeTiled) at run time, so it loads wherever a CUDA 12.8+ driver is present.
The other is plain C++ against the installed torch's headers and libraries, and bears that torch's version in its name: one
that was built against another torch is not taken for this one's.
"""
import importlib.util
import os
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
LIB = os.path.join(HERE, "libbasal200.so")
NVCC_FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a", "-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC",
              "-shared", "-cudart", "static", "--expt-relaxed-constexpr"]


TORCH = os.path.dirname(importlib.util.find_spec("torch").origin)


def torch_version():
    """torch.__version__, without importing torch."""
    spec = importlib.util.spec_from_file_location("basal_b200_torch_version", os.path.join(TORCH, "version.py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod.__version__


TORCH_LIB = os.path.join(HERE, f"libbasal200_torch-{torch_version()}.so")


def sources():
    return sorted(os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith((".cu", ".cuh"))) + \
        [os.path.join(os.path.dirname(HERE), "include", "basal200.h")]


def torch_sources():
    return [os.path.join(CSRC, "step_ops.cpp"), os.path.join(os.path.dirname(HERE), "include", "basal200.h")]


def stale(lib=LIB, of=None):
    if not os.path.exists(lib):
        return True
    t = os.path.getmtime(lib)
    return any(os.path.getmtime(s) > t for s in of or sources())


def build_torch(force=False):
    """Compiles csrc/step_ops.cpp into TORCH_LIB, which finds libbasal200.so beside it."""
    if not force and not stale(TORCH_LIB, torch_sources()):
        return TORCH_LIB
    cuda = os.environ.get("CUDA_HOME", "/usr/local/cuda")
    inc = [f"-I{TORCH}/include", f"-I{TORCH}/include/torch/csrc/api/include", f"-I{cuda}/include"]
    # the system's g++, whose libstdc++ is torch's: a compiler that links its own copy statically gives the library a
    # second set of locales, and formatting an error's text crashes
    subprocess.run(["g++", "-O2", "-std=c++17", "-fPIC", "-shared", *inc, "-o", TORCH_LIB + ".tmp",
                    torch_sources()[0], f"-L{TORCH}/lib", "-lc10", "-lc10_cuda", "-ltorch_cpu", f"-L{HERE}",
                    "-l:libbasal200.so", "-Wl,-rpath,$ORIGIN"], check=True)
    os.replace(TORCH_LIB + ".tmp", TORCH_LIB)
    return TORCH_LIB


def build(force=False, verbose=False):
    """Compiles csrc/basal200.cu into libbasal200.so when a source is newer than the library (or force), then
    TORCH_LIB likewise."""
    if not force and not stale():
        build_torch()
        return LIB
    nvcc = os.environ.get("NVCC", "nvcc")
    cmd = [nvcc, *NVCC_FLAGS, "-o", LIB + ".tmp", os.path.join(CSRC, "basal200.cu")]
    if verbose:
        cmd.insert(1, "-Xptxas=-v")
    subprocess.run(cmd, check=True)
    os.replace(LIB + ".tmp", LIB)
    build_torch(force)
    return LIB


if __name__ == "__main__":
    build(force="--force" in sys.argv, verbose="-v" in sys.argv)
    print(LIB)
