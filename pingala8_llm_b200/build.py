"""Build the in-tree CUDA library pingala8_llm_b200/libpingala8_b200.so for sm_100a (nvcc, no JIT cache) and the Python
module pingala8_llm_b200/_cache_calls.so beside it (g++).

usage: python -m pingala8_llm_b200.build  [--verbose-ptxas]
"""
import argparse
import os
import subprocess
import sys
import sysconfig

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
LIB = os.path.join(HERE, "libpingala8_b200.so")
SOURCES = ["p8_host.cpp", "p8_gguf.cpp", "p8_api.cu", "p8_kernels.cu", "p8_noalloc.cu", "p8_tp.cu", "p8_encode.cu",
           "p8_cache.cu"]
PY_SOURCE = "p8_cache_py.cpp"  # the Python module of the cache operators (host code, against torch's headers)
PY_MODULE = os.path.join(HERE, "_cache_calls.so")
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]


def nvcc():
    for c in (os.environ.get("NVCC"), "/usr/local/cuda/bin/nvcc", "nvcc"):
        if c and (os.path.sep not in c or os.path.exists(c)):
            return c
    return "nvcc"


def build(verbose_ptxas=False, out=LIB, csrc=None, bdir=None):
    csrc = csrc or CSRC
    objs = []
    bdir = bdir or os.path.join(HERE, "_build")
    os.makedirs(bdir, exist_ok=True)
    for s in SOURCES:
        src = os.path.join(csrc, s)
        obj = os.path.join(bdir, s + ".o")
        cmd = [nvcc(), "-std=c++17", "-O3", "-lineinfo", *ARCH, "-Xcompiler", "-fPIC,-O2,-Wall", "-c", src, "-o", obj,
               "-I", csrc, "-I", os.path.join(os.path.dirname(HERE), "include")]
        if s.endswith(".cu") and verbose_ptxas:
            cmd += ["-Xptxas", "-v"]
        print("+", " ".join(cmd), flush=True)
        subprocess.run(cmd, check=True)
        objs.append(obj)
    cmd = [nvcc(), "-shared", *ARCH, *objs, "-o", out, "-lcudart"]
    print("+", " ".join(cmd), flush=True)
    subprocess.run(cmd, check=True)
    return out


def build_py(out=PY_MODULE):
    """The CPython module that checks the cache operators' tensors and fills their argument structures."""
    import torch

    root = os.path.dirname(torch.__file__)
    cuda = os.path.dirname(os.path.dirname(nvcc())) or "/usr/local/cuda"
    inc = [sysconfig.get_paths()["include"], os.path.join(root, "include"), os.path.join(cuda, "include"), os.path.join(os.path.dirname(HERE), "include")]
    cmd = ["g++", "-std=c++17", "-O2", "-Wall", "-fPIC", "-shared", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
           os.path.join(CSRC, PY_SOURCE), "-o", out]
    for i in inc:
        cmd += ["-isystem" if i.startswith(root) else "-I", i]
    cmd += ["-L", os.path.join(root, "lib"), "-ltorch_python", "-ltorch_cpu", "-lc10", "-lc10_cuda"]
    print("+", " ".join(cmd), flush=True)
    subprocess.run(cmd, check=True)
    return out


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--verbose-ptxas", action="store_true")
    a = ap.parse_args()
    build(a.verbose_ptxas)
    build_py()
    sys.exit(0)
