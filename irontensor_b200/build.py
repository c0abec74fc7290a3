"""Builds, in-tree, libirontensor_b200.so with nvcc for sm_100a (cross-compiles without a GPU) and _host_ops.so, the native host
side of the Python ops, with g++ against the installed torch.

    python -m irontensor_b200.build [--force] [--verbose]
"""
import os
import re
import subprocess
import sys

_HERE = os.path.dirname(os.path.abspath(__file__))
_CSRC = os.path.join(_HERE, "csrc")
_OUT = os.path.join(_HERE, "libirontensor_b200.so")
_INC = os.path.join(os.path.dirname(_HERE), "include")
_HOST_SRC = os.path.join(_CSRC, "host_ops.cpp")
_HOST_OUT = os.path.join(_HERE, "_host_ops.so")


_UNITS = ("it_capi.cu", "it_quant.cu")   # translation units of libirontensor_b200.so


def _depends(path, seen=None):
    """`path` and the files of this repository that it includes."""
    seen = set() if seen is None else seen
    if path not in seen and os.path.exists(path):
        seen.add(path)
        with open(path) as f:
            for name in re.findall(r'^\s*#include "([^"]+)"', f.read(), re.M):
                _depends(os.path.normpath(os.path.join(os.path.dirname(path), name)), seen)
    return seen


def _object(unit):
    return os.path.join(_HERE, os.path.splitext(unit)[0] + ".o")


def _newer(out, sources):
    return os.path.exists(out) and all(os.path.getmtime(s) <= os.path.getmtime(out) for s in sources)


def up_to_date():
    return all(_newer(_OUT, _depends(os.path.join(_CSRC, u))) for u in _UNITS)


def _host_up_to_date():
    return os.path.exists(_HOST_OUT) and all(os.path.getmtime(s) <= os.path.getmtime(_HOST_OUT)
                                             for s in (_HOST_SRC, os.path.join(_INC, "irontensor_b200.h")))


def build_host(force=False):
    """_host_ops.so: links libirontensor_b200.so (next to it) and torch's libraries (loaded by `import torch` beforehand)."""
    if not force and _host_up_to_date():
        return _HOST_OUT
    import sysconfig
    import torch
    from torch.utils import cpp_extension as ext
    cmd = [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-shared", "-fPIC", "-fvisibility=hidden", "-Wno-missing-field-initializers",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", "-I" + sysconfig.get_paths()["include"]]
    cmd += ["-isystem" + p for p in ext.include_paths() + ["/usr/local/cuda/include"]]
    cmd += [_HOST_SRC, "-o", _HOST_OUT, "-L" + _HERE, "-l:libirontensor_b200.so", "-Wl,-rpath,$ORIGIN"]
    cmd += ["-L" + p for p in ext.library_paths()] + ["-lc10", "-ltorch_cpu", "-ltorch_python", "-lc10_cuda", "-ltorch_cuda"]
    subprocess.run(cmd, check=True)
    return _HOST_OUT


def build(force=False, verbose=False):
    if not force and up_to_date():
        build_host()
        return _OUT
    nvcc = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")
    arch = ["-gencode", "arch=compute_100a,code=sm_100a"]
    flags = [*arch, "-lineinfo", "-O3", "-std=c++17", "-Xcompiler", "-fPIC"]
    if verbose:
        flags = ["-Xptxas", "-v"] + flags
    running = []   # the units that changed, side by side
    for unit in _UNITS:
        src, obj = os.path.join(_CSRC, unit), _object(unit)
        if force or not _newer(obj, _depends(src)):
            cmd = [nvcc, *flags, "-c", "-o", obj + ".new", src]
            running.append((cmd, obj, subprocess.Popen(cmd)))
    codes = [p.wait() for _, _, p in running]
    for (cmd, obj, _), rc in zip(running, codes):
        if rc != 0:
            raise subprocess.CalledProcessError(rc, cmd)
        os.replace(obj + ".new", obj)
    subprocess.run([nvcc, *arch, "-shared", "-o", _OUT, *[_object(u) for u in _UNITS]], check=True)
    build_host(force)
    return _OUT


if __name__ == "__main__":
    build(force="--force" in sys.argv, verbose="--verbose" in sys.argv)
    print(_OUT)
