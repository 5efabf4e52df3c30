"""Build librw4.so, the RW4 C-ABI library, for sm_100a with nvcc (in-tree, no JIT cache).

    python -m rocketllm_b200.csrc.build          # or: python rocketllm_b200/csrc/build.py

Every .cu / .cpp file in this folder is compiled with
``-gencode arch=compute_100a,code=sm_100a -lineinfo -O3`` and linked into
``rocketllm_b200/librw4.so`` next to the package, so the library travels with the source tree.
``binding/rw4_native.cpp`` (the host fast path of the 8-bit operators' Python entry points) is
compiled against torch's headers and linked into ``rocketllm_b200/_rw4_native.so``, which loads
``librw4.so`` from its own folder; where torch, Python's headers or g++ are missing it is left out.
Rebuilds only when a source or header is newer than the library (``_rw4_native.so`` also when torch
or Python is another one).
"""
import glob
import os
import shutil
import subprocess
import sys
import sysconfig

HERE = os.path.dirname(os.path.abspath(__file__))
PKG = os.path.dirname(HERE)
ROOT = os.path.dirname(PKG)
LIB = os.path.join(PKG, "librw4.so")
NATIVE_SRC = os.path.join(HERE, "binding", "rw4_native.cpp")
NATIVE = os.path.join(PKG, "_rw4_native.so")
BUILD_DIR = os.path.join(PKG, "_build")
NATIVE_STAMP = os.path.join(BUILD_DIR, "rw4_native.against")   # the torch and Python it was built for
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]


def nvcc():
    cand = os.path.join(os.environ.get("CUDA_HOME", "/usr/local/cuda"), "bin", "nvcc")
    return cand if os.path.exists(cand) else "nvcc"


def sources():
    return sorted(glob.glob(os.path.join(HERE, "*.cu")) + glob.glob(os.path.join(HERE, "*.cpp")))


def headers():
    return (glob.glob(os.path.join(HERE, "*.cuh")) + glob.glob(os.path.join(HERE, "*.h"))
            + glob.glob(os.path.join(ROOT, "include", "*.h")))


def stale(target, deps):
    if not os.path.exists(target):
        return True
    t = os.path.getmtime(target)
    return any(os.path.getmtime(d) > t for d in deps)


def build(verbose=False, force=False, extra=()):
    os.makedirs(BUILD_DIR, exist_ok=True)
    objs = []
    hdrs = headers()
    for src in sources():
        obj = os.path.join(BUILD_DIR, os.path.basename(src) + ".o")
        objs.append(obj)
        if not force and not stale(obj, [src] + hdrs):
            continue
        cmd = [nvcc(), *ARCH, "-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC",
               "-I", os.path.join(ROOT, "include"), "-c", src, "-o", obj, *extra]
        if src.endswith(".cpp"):
            cmd[1:1] = ["-x", "cu"]
        if verbose:
            cmd.insert(1, "-Xptxas=-v")
            print(" ".join(cmd), flush=True)
        subprocess.run(cmd, check=True)
    if force or stale(LIB, objs):
        cmd = [nvcc(), *ARCH, "-shared", "-o", LIB, *objs, "-lcuda", "-lcudart"]
        if verbose:
            print(" ".join(cmd), flush=True)
        subprocess.run(cmd, check=True)
    build_native(verbose, force)
    return LIB


def native_missing():
    """What ``_rw4_native.so`` needs and this machine lacks (empty: it can be built)."""
    missing = [] if shutil.which("g++") else ["g++"]
    if not os.path.exists(os.path.join(sysconfig.get_paths()["include"], "Python.h")):
        missing.append("Python.h")
    try:
        import torch  # noqa: F401
    except ImportError:
        missing.append("torch")
    return missing


def build_native(verbose=False, force=False):
    """``_rw4_native.so``: host C++ only (no device code), against the installed torch and Python;
    built again when either is another one.  Without its prerequisites it is left out, with a line
    that says so: the library does not need it (the Python entry points call it through ctypes)."""
    missing = native_missing()
    if missing:
        print(f"{os.path.basename(NATIVE)} left out: no {', '.join(missing)} here", flush=True)
        return
    import torch
    against = f"torch {torch.__version__}, {sys.implementation.cache_tag}"
    try:
        with open(NATIVE_STAMP) as f:
            same = f.read() == against
    except OSError:
        same = False
    if same and not force and not stale(NATIVE, [NATIVE_SRC, os.path.join(ROOT, "include",
                                                                          "rw4.h")]):
        return
    troot = os.path.dirname(torch.__file__)
    cuda = os.environ.get("CUDA_HOME", "/usr/local/cuda")
    abi = int(torch.compiled_with_cxx11_abi())
    cmd = ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", f"-D_GLIBCXX_USE_CXX11_ABI={abi}",
           f'-DRW4_TORCH_VERSION="{torch.__version__}"',
           "-I", sysconfig.get_paths()["include"], "-I", os.path.join(troot, "include"),
           "-I", os.path.join(troot, "include", "torch", "csrc", "api", "include"),
           "-I", os.path.join(cuda, "include"), "-I", os.path.join(ROOT, "include"),
           NATIVE_SRC, "-o", NATIVE, "-L", os.path.join(troot, "lib"), "-ltorch_python",
           "-ltorch_cpu", "-ltorch_cuda", "-lc10", "-lc10_cuda", "-L", PKG, "-lrw4",
           "-Wl,-rpath,$ORIGIN"]
    if verbose:
        print(" ".join(cmd), flush=True)
    subprocess.run(cmd, check=True)
    os.makedirs(BUILD_DIR, exist_ok=True)
    with open(NATIVE_STAMP, "w") as f:
        f.write(against)


if __name__ == "__main__":
    build(verbose="-v" in sys.argv, force="-f" in sys.argv)
    print(LIB)
