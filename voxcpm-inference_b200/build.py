"""Builds libvxb.so (CUDA kernels + C ABI + C++ host API) for sm_100a and, where
torch and Python's headers are installed, the Python module _vxb_native.so
(torch tensors to the C ABI), in-tree.

    python voxcpm-inference_b200/build.py [-v]

Objects go to voxcpm-inference_b200/_build/, the libraries to
voxcpm-inference_b200/lib/.  Only files whose sources (or shared
headers, or for the module torch) changed are recompiled.
"""
from __future__ import annotations

import concurrent.futures as cf
import glob
import importlib.util
import os
import subprocess
import sys
import sysconfig

PKG = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(PKG)
CSRC = os.path.join(PKG, "csrc")
BUILD = os.path.join(PKG, "_build")
LIB = os.path.join(PKG, "lib", "libvxb.so")
NATIVE = os.path.join(PKG, "lib", "_vxb_native.so")
NVCC = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
INC = ["-I" + os.path.join(ROOT, "include"), "-I" + CSRC, "-I" + os.path.join(PKG, "include")]


def _sources():
    cu = sorted(glob.glob(os.path.join(CSRC, "*.cu")))
    cpp = sorted(glob.glob(os.path.join(CSRC, "*.cpp")) + glob.glob(os.path.join(CSRC, "host", "*.cpp")))
    return cu, cpp


def _torch():
    """torch's folder, or None where the Python module cannot be built (a C or C++
    caller of libvxb.so needs neither torch nor Python's headers)."""
    spec = importlib.util.find_spec("torch")
    path = spec.submodule_search_locations[0] if spec else ""
    needed = [os.path.join(path, "include", "c10", "cuda", "CUDAStream.h"),
              os.path.join(sysconfig.get_paths()["include"], "Python.h")]
    return path if all(os.path.exists(f) for f in needed) else None


def _made_for(torch):
    """What the module is compiled against besides this repository's sources."""
    with open(os.path.join(torch, "version.py")) as f:
        return sys.version + "\n" + torch + "\n" + f.read()


def _headers():
    hs = glob.glob(os.path.join(CSRC, "**", "*.cuh"), recursive=True)
    hs += glob.glob(os.path.join(CSRC, "**", "*.h"), recursive=True)
    hs += glob.glob(os.path.join(ROOT, "include", "*.h"))
    hs += glob.glob(os.path.join(PKG, "include", "**", "*.h"), recursive=True)
    return hs


def _stale(obj, src, hdr_mtime):
    return not os.path.exists(obj) or os.path.getmtime(obj) < max(os.path.getmtime(src), hdr_mtime)


def _run(cmd, verbose):
    if verbose:
        print(" ".join(cmd), flush=True)
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"build failed: {' '.join(cmd)}\n{r.stdout}\n{r.stderr}")
    return r.stdout + r.stderr


def build(verbose: bool = False) -> str:
    os.makedirs(BUILD, exist_ok=True)
    os.makedirs(os.path.dirname(LIB), exist_ok=True)
    cu, cpp = _sources()
    hdr_mtime = max([os.path.getmtime(h) for h in _headers()] + [os.path.getmtime(__file__)])
    jobs, objs = [], []
    for s in cu:
        o = os.path.join(BUILD, os.path.basename(s) + ".o")
        objs.append(o)
        if _stale(o, s, hdr_mtime):
            jobs.append([NVCC, *ARCH, "-lineinfo", "-O3", "-std=c++17", "-Xcompiler", "-fPIC,-fvisibility=hidden",
                         *INC, "-c", s, "-o", o])
    for s in cpp:
        o = os.path.join(BUILD, os.path.basename(s) + ".o")
        objs.append(o)
        if _stale(o, s, hdr_mtime):
            jobs.append(["g++", "-O2", "-std=c++17", "-fPIC", "-fvisibility=hidden", "-Wall",
                         "-I/usr/local/cuda/include", *INC, "-c", s, "-o", o])
    torch, bind_jobs = _torch(), []
    bind, bind_obj = os.path.join(CSRC, "bind", "native.cpp"), os.path.join(BUILD, "native.cpp.o")
    stamp = bind_obj + ".for"
    if torch is None:
        print("torch or Python.h not found: libvxb.so only, without the Python module " + os.path.basename(NATIVE),
              file=sys.stderr)
    else:
        inc = os.path.join(torch, "include")
        abi = os.path.join(ROOT, "include", "vxb.h")
        same = os.path.exists(stamp) and open(stamp).read() == _made_for(torch)
        if not same or _stale(bind_obj, bind, max(os.path.getmtime(abi), os.path.getmtime(__file__))):
            bind_jobs.append(["g++", "-O2", "-std=c++17", "-fPIC", "-fvisibility=hidden", "-Wall", "-I" + inc,
                              "-I" + os.path.join(inc, "torch", "csrc", "api", "include"),
                              "-I" + sysconfig.get_paths()["include"], "-I/usr/local/cuda/include", *INC, "-c", bind,
                              "-o", bind_obj])
    with cf.ThreadPoolExecutor(max_workers=os.cpu_count() or 4) as ex:
        for out in ex.map(lambda c: _run(c, verbose), jobs + bind_jobs):
            if verbose and out.strip():
                print(out)
    if jobs or not os.path.exists(LIB):
        _run([NVCC, *ARCH, "-shared", "-cudart", "static", "-o", LIB, *objs, "-lpthread", "-ldl", "-lrt"], verbose)
    if torch is not None and (bind_jobs or not os.path.exists(NATIVE)):
        lib = os.path.join(torch, "lib")
        _run(["g++", "-shared", "-o", NATIVE, bind_obj, "-L" + os.path.dirname(LIB), "-lvxb", "-L" + lib,
              "-ltorch_python", "-ltorch_cpu", "-lc10_cuda", "-lc10", "-Wl,-rpath,$ORIGIN", "-Wl,-rpath," + lib],
             verbose)
        with open(stamp, "w") as f:
            f.write(_made_for(torch))
    return LIB


if __name__ == "__main__":
    print(build(verbose="-v" in sys.argv))
