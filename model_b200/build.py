"""Build the memory-layer CUDA library in-tree (``model_b200/libmemlayer.so``).

Every ``csrc/*.cu`` file is compiled for sm_100a only
(``-gencode arch=compute_100a,code=sm_100a``) and linked into one shared
library that exports the C ABI of ``include/memlayer.h``.  nvcc
cross-compiles without a GPU, so this runs on any machine with CUDA 12.9.
``csrc/fast_calls.cpp``, the training operators' calls from torch tensors, is
compiled beside it against this interpreter and its torch, again whenever one
of them or the command changes.  Without it (no host compiler, no headers) the
operators go over ctypes, so a failure there is a warning.
"""

from __future__ import annotations

import concurrent.futures as cf
import glob
import os
import subprocess
import sys
import sysconfig

PKG = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(PKG)
CSRC = os.path.join(PKG, "csrc")
INCLUDE = os.path.join(ROOT, "include")
BUILD = os.path.join(ROOT, "_build")
LIB = os.path.join(PKG, "libmemlayer.so")
FAST = os.path.join(PKG, "_fast" + sysconfig.get_config_var("EXT_SUFFIX"))
FAST_STAMP = os.path.join(BUILD, "fast_calls.stamp")   # what FAST was built with

NVCC = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
FLAGS = ["-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC", "--expt-relaxed-constexpr",
         "-I", INCLUDE, "-I", CSRC]


def _stale(obj: str, deps) -> bool:
    if not os.path.exists(obj):
        return True
    t = os.path.getmtime(obj)
    return any(os.path.getmtime(d) > t for d in deps)


def _fast_command():
    """The compiler's command for the extension module, and the module's dependencies."""
    import torch
    tdir = os.path.dirname(torch.__file__)
    tinc, cuda = os.path.join(tdir, "include"), os.path.dirname(os.path.dirname(NVCC))
    src = os.path.join(CSRC, "fast_calls.cpp")
    cmd = [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-fPIC", "-shared",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
           f'-DMEMLAYER_TORCH_VERSION="{torch.__version__}"', src, "-o", FAST, "-I", INCLUDE,
           "-I", tinc, "-I", os.path.join(tinc, "torch", "csrc", "api", "include"),
           "-I", os.path.join(cuda, "include"), "-I", sysconfig.get_paths()["include"],
           "-L", PKG, "-l:" + os.path.basename(LIB), "-L", os.path.join(tdir, "lib"), "-lc10", "-lc10_cuda",
           "-ltorch_cpu", "-ltorch_python", "-Wl,-rpath,$ORIGIN"]
    return cmd, [src, os.path.join(INCLUDE, "memlayer.h")]


def build_fast() -> bool:
    """The extension module, where it is not what this torch, source and command give; False: not built."""
    cmd, deps = _fast_command()
    stamp = "\n".join([sys.version, *cmd])           # the command names torch's version and folder
    try:
        with open(FAST_STAMP) as f:
            same = f.read() == stamp
    except OSError:
        same = False
    if same and not _stale(FAST, deps):
        return True
    if os.path.exists(FAST):
        os.remove(FAST)                              # one of another torch must not be loaded
    try:
        r = subprocess.run(cmd, capture_output=True, text=True)
        failed = None if r.returncode == 0 else f"{r.stdout}\n{r.stderr}"
    except OSError as e:
        failed = str(e)
    if failed is not None:
        print(f"warning: {os.path.basename(FAST)} is not built, the training operators' calls go over ctypes "
              f"({' '.join(cmd)}):\n{failed}", file=sys.stderr)
        return False
    with open(FAST_STAMP, "w") as f:
        f.write(stamp)
    return True


def build(verbose: bool = False, ptxas_verbose: bool = False) -> str:
    os.makedirs(BUILD, exist_ok=True)
    sources = sorted(glob.glob(os.path.join(CSRC, "*.cu")))
    headers = glob.glob(os.path.join(CSRC, "*.cuh")) + glob.glob(os.path.join(INCLUDE, "*.h"))
    objs, jobs = [], []
    for src in sources:
        obj = os.path.join(BUILD, os.path.basename(src)[:-3] + ".o")
        objs.append(obj)
        if _stale(obj, [src, *headers]):
            cmd = [NVCC, *ARCH, *FLAGS, "-c", src, "-o", obj]
            if ptxas_verbose:
                cmd += ["-Xptxas", "-v"]
            jobs.append(cmd)

    def run(cmd):
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"{os.path.basename(cmd[0])} failed ({' '.join(cmd)}):\n{r.stdout}\n{r.stderr}")
        return r.stdout + r.stderr

    with cf.ThreadPoolExecutor(max_workers=min(8, os.cpu_count() or 1)) as ex:
        for out in ex.map(run, jobs):
            if verbose and out.strip():
                print(out)
    if jobs or not os.path.exists(LIB):
        run([NVCC, *ARCH, "-shared", "-o", LIB, *objs, "-lcudart_static", "-Xlinker",
             "-rpath=/usr/local/cuda/lib64", "-lrt", "-ldl", "-lpthread"])
    build_fast()
    # the XLA FFI handlers of the JAX binding, where JAX is installed
    from model_b200 import jax_ffi
    jax_ffi.build(verbose=verbose)
    return LIB


if __name__ == "__main__":
    print(build(verbose=True, ptxas_verbose="-v" in sys.argv))
