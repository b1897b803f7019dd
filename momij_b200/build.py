"""Builds libmomij_moe.so in-tree (momij_b200/lib/) for sm_100a with nvcc, and
_momij_ops.so beside it (the Python entry of the attn and head operators).

Each .cu under csrc/ is compiled separately (parallel), then linked into one
shared library with the CUDA runtime linked statically, so the library does
not depend on which libcudart the host process has loaded.  Usage:
``python -m momij_b200.build [-j N] [--verbose-ptxas]``.
"""
from __future__ import annotations

import argparse
import concurrent.futures as cf
import os
import shutil
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
CSRC = os.path.join(HERE, "csrc")
OBJ = os.path.join(HERE, "_build")
LIB_DIR = os.path.join(HERE, "lib")
LIB = os.path.join(LIB_DIR, "libmomij_moe.so")
SOURCES = ["route.cu", "gemv.cu", "layer.cu", "token.cu", "decode.cu", "block.cu", "prefill.cu", "ep.cu", "ep_host.cu", "misc.cu",
           "api.cu", "noalloc.cu", "kvcache.cu", "attn.cu", "attn_prefill.cu", "qmm4.cu", "qmm4_tc.cu", "logits.cu"]

ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]


def nvcc() -> str:
    for cand in (os.environ.get("NVCC"), "/usr/local/cuda/bin/nvcc", shutil.which("nvcc")):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found")


def _flags(verbose_ptxas: bool) -> list[str]:
    f = ARCH + ["-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC,-O3",
                "-I", os.path.join(ROOT, "include"), "-I", CSRC, "--expt-relaxed-constexpr",
                "-ccbin", "/usr/bin/g++"]
    if verbose_ptxas:
        f += ["-Xptxas", "-v"]
    return f


def _compile(src: str, verbose_ptxas: bool) -> str:
    out = os.path.join(OBJ, os.path.splitext(src)[0] + ".o")
    path = os.path.join(CSRC, src)
    deps = [path] + [os.path.join(CSRC, h) for h in os.listdir(CSRC) if h.endswith(".cuh")]
    deps.append(os.path.join(ROOT, "include", "momij_moe.h"))
    if (not verbose_ptxas and os.path.exists(out)
            and os.path.getmtime(out) >= max(os.path.getmtime(d) for d in deps)):
        return out
    cmd = [nvcc()] + _flags(verbose_ptxas) + ["-c", path, "-o", out]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"nvcc failed for {src}:\n{r.stderr}")
    if verbose_ptxas:
        sys.stderr.write(r.stderr)
    return out


def _bind_is_current(out: str, deps: list[str], stamp: str, made_with: str) -> bool:
    """Whether ``out`` is newer than its sources and was built against this torch and
    Python (``stamp`` holds what the last build used): another's headers may lay
    tensors out differently."""
    if not os.path.exists(out) or os.path.getmtime(out) < max(os.path.getmtime(d) for d in deps):
        return False
    if not os.path.exists(stamp):
        return False
    with open(stamp) as f:
        return f.read() == made_with


def _bind() -> str:
    """_momij_ops.so: the Python entry of the attn and head operators (a CPython
    module over torch's tensors; libmomij_moe.so itself needs neither)."""
    import sysconfig

    import torch
    src = os.path.join(CSRC, "bind.cpp")
    out = os.path.join(LIB_DIR, "_momij_ops.so")
    deps = [src, os.path.join(ROOT, "include", "momij_moe.h")]
    stamp, made_with = os.path.join(OBJ, "bind.stamp"), f"{torch.__version__} {torch.version.cuda} {torch.__file__} {sys.version}"
    if _bind_is_current(out, deps, stamp, made_with):
        return out
    inc, lib = os.path.join(os.path.dirname(torch.__file__), "include"), os.path.join(os.path.dirname(torch.__file__), "lib")
    cuda = os.path.dirname(os.path.dirname(nvcc()))
    cmd = ["/usr/bin/g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden", src, "-o", out,
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", "-I", os.path.join(ROOT, "include"),
           "-isystem", inc, "-isystem", os.path.join(inc, "torch", "csrc", "api", "include"),
           "-isystem", sysconfig.get_paths()["include"], "-isystem", os.path.join(cuda, "include"),
           "-L", lib, "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch_cuda", "-ltorch_python"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"g++ failed for bind.cpp:\n{r.stderr}")
    with open(stamp, "w") as f:
        f.write(made_with)
    return out


def build(jobs: int = 4, verbose_ptxas: bool = False) -> str:
    os.makedirs(OBJ, exist_ok=True)
    os.makedirs(LIB_DIR, exist_ok=True)
    with cf.ThreadPoolExecutor(max_workers=jobs) as ex:
        bound = ex.submit(_bind)
        objs = list(ex.map(lambda s: _compile(s, verbose_ptxas), SOURCES))
        bound.result()
    if (not os.path.exists(LIB) or
            os.path.getmtime(LIB) < max(os.path.getmtime(o) for o in objs)):
        cmd = [nvcc()] + ARCH + ["-shared", "-o", LIB] + objs + ["-cudart", "static", "-ldl",
                                                                  "-ccbin", "/usr/bin/g++"]
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"link failed:\n{r.stderr}")
    return LIB


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("-j", type=int, default=4)
    ap.add_argument("--verbose-ptxas", action="store_true")
    args = ap.parse_args()
    print(build(args.j, args.verbose_ptxas))
