"""Builds librocal_b200.so (CUDA kernels + C-ABI + host pipeline) in-tree for sm_100a, and _head.so (the torch binding of the
head operators, g++ against the installed torch).

    python -m rocal_b200.build [--force] [--verbose] [--debug-bounds]

--debug-bounds builds librocal_b200_bounds.so instead: the same sources with RB200_DEBUG_BOUNDS defined, in which the
kernels check every sample's source rectangle and every staging copy against the arena size the caller states and
report through the status word (include/rb200_kernels.h, "Sizes and the bounds-checking build"). Load it by setting
RB200_LIBRARY to its path.

nvcc cross-compiles without a GPU. The library links the CUDA runtime statically, so it loads
in any process whether or not another CUDA runtime (e.g. torch's) is already present.
"""
import glob
import os
import subprocess
import sys

PKG = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(PKG)
CSRC = os.path.join(PKG, "csrc")
LIB = os.path.join(PKG, "librocal_b200.so")
OBJ_DIR = os.path.join(PKG, "build")

NVCC = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
COMMON = ["-O3", "-std=c++17", "-lineinfo", "-Xcompiler", "-fPIC,-fvisibility=hidden,-Wall",
          "-I" + os.path.join(ROOT, "include"), "-I" + os.path.join(CSRC, "kernels"),
          "-I" + os.path.join(CSRC, "host")]


def sources():
    return sorted(glob.glob(os.path.join(CSRC, "kernels", "*.cu")) + glob.glob(os.path.join(CSRC, "host", "*.cpp")))


def headers():
    return (glob.glob(os.path.join(CSRC, "kernels", "*.cuh")) + glob.glob(os.path.join(CSRC, "host", "*.h")) +
            glob.glob(os.path.join(ROOT, "include", "*.h")))


HEAD_SRC = os.path.join(CSRC, "torch", "head.cpp")
HEAD_LIB = os.path.join(PKG, "_head.so")


HEAD_STAMP = os.path.join(OBJ_DIR, "_head.stamp")     # what _head.so was compiled against


def head_versions():
    """The torch and Python that _head.so has to be compiled against, or None without a torch that has CUDA. (torch is not
    imported: that takes longer than looking whether anything has to be built.)"""
    import importlib.util
    import re
    spec = importlib.util.find_spec("torch")
    if spec is None or not os.path.exists(os.path.join(os.path.dirname(spec.origin), "lib", "libc10_cuda.so")):
        return None
    with open(os.path.join(os.path.dirname(spec.origin), "version.py")) as f:     # there without a package's metadata, too
        version = re.search(r"__version__\s*=\s*['\"]([^'\"]+)", f.read())
    return "torch %s, Python %d.%d" % ((version.group(1) if version else "of no version",) + sys.version_info[:2])


def head_stamp():
    """The versions, and on further lines where they lie."""
    import importlib.util
    return "\n".join([head_versions(), os.path.dirname(importlib.util.find_spec("torch").origin), sys.prefix, NVCC]) + "\n"


def head_command():
    """The compiler call that makes _head.so, the torch binding of the head operators. It calls the library through
    addresses it is given at import, so it does not link to it."""
    import sysconfig

    import torch
    root = os.path.join(os.path.dirname(torch.__file__))
    cuda = os.path.dirname(os.path.dirname(NVCC))
    includes = [os.path.join(ROOT, "include"), os.path.join(root, "include"), os.path.join(root, "include", "torch", "csrc", "api", "include"),
                os.path.join(cuda, "include"), sysconfig.get_paths()["include"]]
    libs = os.path.join(root, "lib")
    return (["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden", "-w", "-DTORCH_EXTENSION_NAME=_head",
             "-D_GLIBCXX_USE_CXX11_ABI=%d" % int(torch._C._GLIBCXX_USE_CXX11_ABI)] + ["-isystem" + i for i in includes[1:]] +
            ["-I" + includes[0], HEAD_SRC, "-o", HEAD_LIB, "-L" + libs, "-ltorch", "-ltorch_cpu", "-ltorch_python", "-lc10", "-lc10_cuda",
             "-Wl,-rpath," + libs])


def build_head(force=False):
    """Starts the build of _head.so where it is out of date - with its sources, or with the torch or the Python that it was compiled
    against; returns the process to wait for, or None. Without a torch that has CUDA there is no binding to build: the library
    itself does not need one."""
    if head_versions() is None:
        sys.stderr.write("rocal_b200: no torch with CUDA is installed, the torch binding of the head operators is not built\n")
        return None
    newest = max(os.path.getmtime(f) for f in (HEAD_SRC, os.path.join(ROOT, "include", "rb200_kernels.h"), __file__))
    stamp = ""
    if os.path.exists(HEAD_STAMP):
        with open(HEAD_STAMP) as f:
            stamp = f.read()
    if not force and os.path.exists(HEAD_LIB) and os.path.getmtime(HEAD_LIB) > newest and stamp == head_stamp():
        return None
    return subprocess.Popen(head_command(), stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)


LIB_BOUNDS = os.path.join(PKG, "librocal_b200_bounds.so")


def build(force=False, verbose=False, debug_bounds=False):
    lib = LIB_BOUNDS if debug_bounds else LIB
    obj_dir = OBJ_DIR + ("_bounds" if debug_bounds else "")
    defines = ["-DRB200_DEBUG_BOUNDS"] if debug_bounds else []
    os.makedirs(obj_dir, exist_ok=True)
    hdr_time = max([os.path.getmtime(h) for h in headers()] + [os.path.getmtime(__file__)])
    objs, procs = [], []
    head = None if debug_bounds else build_head(force)
    for src in sources():
        obj = os.path.join(obj_dir, os.path.basename(src) + ".o")
        objs.append(obj)
        if (not force and os.path.exists(obj) and os.path.getmtime(obj) > os.path.getmtime(src)
                and os.path.getmtime(obj) > hdr_time):
            continue
        cmd = [NVCC] + ARCH + COMMON + defines + (["-Xptxas", "-v"] if verbose else []) + ["-x", "cu", "-c", src, "-o", obj]
        procs.append((src, subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)))
    failed = False
    for src, p in procs:
        out, _ = p.communicate()
        if p.returncode != 0 or verbose:
            sys.stderr.write(out)
        if p.returncode != 0:
            failed = True
            sys.stderr.write("nvcc failed for %s\n" % src)
    if head is not None:
        out, _ = head.communicate()
        if head.returncode != 0:
            failed = True
            sys.stderr.write(out + "g++ failed for %s\n" % HEAD_SRC)
        else:
            with open(HEAD_STAMP, "w") as f:
                f.write(head_stamp())
    if failed:
        raise RuntimeError("rocal_b200: nvcc build failed")
    if procs or force or not os.path.exists(lib):
        cmd = [NVCC] + ARCH + ["-shared", "-o", lib] + objs + ["-Xlinker", "--exclude-libs,ALL", "-lpthread"]
        subprocess.run(cmd, check=True)
    return lib


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="--verbose" in sys.argv, debug_bounds="--debug-bounds" in sys.argv))
