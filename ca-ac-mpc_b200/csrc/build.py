"""Build libilqr_b200.so (the C-ABI solver library) in-tree for sm_100a.

    python ca-ac-mpc_b200/csrc/build.py [--verbose]

Compiles every .cu file in this directory with nvcc for sm_100a
(-gencode arch=compute_100a,code=sm_100a, -lineinfo, -fmad=false so the model
arithmetic rounds like the reference's elementwise torch ops; FILE_FLAGS adds
per-file options) and links them
into ca-ac-mpc_b200/libilqr_b200.so, then the torch binding of the calls that
take lists of tensors (binding/ilqr_torch.cpp) with g++ into
ca-ac-mpc_b200/ilqr_torch.so, a Python module. The library needs no torch: where
what the binding is built with is not there, it is left out with a message, and
its calls say so. Objects are rebuilt only when a
source or header is newer than the object (make-style), in parallel, the binding
also when torch or Python is another than it was built with.
"""

from __future__ import annotations

import argparse
import concurrent.futures as cf
import glob
import os
import shutil
import subprocess
import sys
import sysconfig

HERE = os.path.dirname(os.path.abspath(__file__))
PKG = os.path.dirname(HERE)
ROOT = os.path.dirname(PKG)
OBJ_DIR = os.path.join(ROOT, "_build", "obj")
LIB = os.path.join(PKG, "libilqr_b200.so")
PROBE_LIB = os.path.join(PKG, "libilqr_probe.so")
PROBE_SRC = os.path.join(HERE, "probe", "fma_probe.cu")
BINDING_SRC = os.path.join(HERE, "binding", "ilqr_torch.cpp")
BINDING_FILES = [BINDING_SRC, os.path.join(ROOT, "include", "ilqr_b200.h"), os.path.join(HERE, "ilqr_overlap.h")]
BINDING = os.path.join(PKG, "ilqr_torch.so")
NVCC = os.environ.get("NVCC", "nvcc")
CXX = "g++"  # as nvcc takes it (torch and the binding share one libstdc++)
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
FLAGS = ["-O3", "-std=c++17", "-lineinfo", "-fmad=false", "-Xcompiler", "-fPIC,-O2",
         "-I", os.path.join(ROOT, "include"), "-I", HERE]
# Per-file additions. The FastMPC numerics kernels restate a build compiled
# with --use_fast_math, whose divisions are the approximate (2-ulp) kind; they
# use that division too (at B = 16384 the solve takes 5.4 ms instead of 8.5 ms
# with IEEE division, inside the same parity bars).
FILE_FLAGS = {"ilqr_fastmpc.cu": ["-prec-div=false"]}


def _newer(src_files, target):
    if not os.path.exists(target):
        return True
    t = os.path.getmtime(target)
    return any(os.path.getmtime(s) > t for s in src_files)


def binding_needs() -> list:
    """What the torch binding is built with and is not here."""
    if shutil.which(CXX) is None:
        return [CXX]
    try:
        import torch
    except ImportError:
        return ["torch"]
    at = os.path.dirname(torch.__file__)
    files = [os.path.join(at, "include", "torch", "csrc", "autograd", "python_variable.h"),
             os.path.join(at, "include", "c10", "cuda", "CUDAGuard.h"),
             os.path.join(_cuda_home(), "include", "cuda_runtime_api.h"),
             os.path.join(sysconfig.get_paths()["include"], "Python.h"),
             *(os.path.join(at, "lib", f"lib{n}.so") for n in TORCH_LIBS)]
    return [f for f in files if not os.path.exists(f)]


def _cuda_home() -> str:
    return os.environ.get("CUDA_HOME", "/usr/local/cuda")


TORCH_LIBS = ("torch_python", "torch", "torch_cpu", "torch_cuda", "c10", "c10_cuda")


def build_binding() -> str:
    """The torch binding, against the torch that is importable here and the
    C-ABI library beside it."""
    import torch
    at = os.path.dirname(torch.__file__)
    inc = [os.path.join(at, "include"), os.path.join(at, "include", "torch", "csrc", "api", "include"),
           os.path.join(_cuda_home(), "include"), sysconfig.get_paths()["include"], os.path.join(ROOT, "include")]
    cmd = [CXX, "-std=c++20", "-O2", "-fPIC", "-shared",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", *[f"-I{d}" for d in inc],
           BINDING_SRC, "-o", BINDING, f"-L{os.path.join(at, 'lib')}", *[f"-l{n}" for n in TORCH_LIBS],
           f"-L{PKG}", "-l:libilqr_b200.so", "-Wl,-rpath,$ORIGIN"]
    # what it was built against: files of another torch may be older than it
    made = "\n".join([torch.__version__, str(torch.version.git_version), sys.version, *cmd])
    stamp = os.path.join(OBJ_DIR, "ilqr_torch.stamp")
    if _newer(BINDING_FILES, BINDING) or not os.path.exists(stamp) or open(stamp).read() != made:
        os.makedirs(OBJ_DIR, exist_ok=True)
        if os.path.exists(stamp):
            os.remove(stamp)  # a build that is interrupted leaves none
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError("torch binding build failed:\n" + r.stdout + r.stderr)
        with open(stamp, "w") as f:
            f.write(made)
    return BINDING


def build(verbose: bool = False) -> str:
    os.makedirs(OBJ_DIR, exist_ok=True)
    sources = sorted(glob.glob(os.path.join(HERE, "*.cu")))
    headers = sorted(glob.glob(os.path.join(HERE, "*.cuh")) + glob.glob(os.path.join(HERE, "*.h"))
                     + glob.glob(os.path.join(ROOT, "include", "*.h")))
    jobs = []
    objs = []
    for src in sources:
        obj = os.path.join(OBJ_DIR, os.path.basename(src).replace(".cu", ".o"))
        objs.append(obj)
        if _newer([src, os.path.abspath(__file__)] + headers, obj):
            cmd = [NVCC, *ARCH, *FLAGS, *FILE_FLAGS.get(os.path.basename(src), []), "-c", src, "-o", obj]
            if verbose:
                cmd.insert(1, "-Xptxas=-v")
            jobs.append(cmd)

    def run(cmd):
        r = subprocess.run(cmd, capture_output=True, text=True)
        return cmd, r

    failed = False
    with cf.ThreadPoolExecutor(max_workers=max(1, min(len(jobs), os.cpu_count() or 1))) as ex:
        for cmd, r in ex.map(run, jobs):
            out = (r.stdout + r.stderr).strip()
            if r.returncode != 0:
                failed = True
                sys.stderr.write(" ".join(cmd) + "\n" + out + "\n")
            elif verbose and out:
                print(out)
    if failed:
        raise RuntimeError("nvcc failed")
    if jobs or _newer(objs, LIB):
        link = [NVCC, *ARCH, "-shared", "-o", LIB, *objs, "-lcudart_static", "-ldl", "-lrt", "-lpthread"]
        r = subprocess.run(link, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError("link failed:\n" + r.stdout + r.stderr)
    # FP32 FMA throughput probe used by the benchmark's roofline (separate
    # library: measurement only).
    if _newer([PROBE_SRC], PROBE_LIB):
        cmd = [NVCC, *ARCH, "-O3", "-Xcompiler", "-fPIC", "-shared", PROBE_SRC, "-o", PROBE_LIB]
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError("probe build failed:\n" + r.stdout + r.stderr)
    missing = binding_needs()
    if missing:
        if os.path.exists(BINDING) and _newer(BINDING_FILES, BINDING):
            os.remove(BINDING)  # of an earlier source
        print("the torch binding of the gradient norms and clipping was not built, for want of: " + ", ".join(missing),
              file=sys.stderr)
    else:
        build_binding()
    return LIB


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--verbose", action="store_true")
    a = ap.parse_args()
    print(build(verbose=a.verbose))
