"""Build the in-tree C-ABI library ``logkv_b200/liblogkv_b200.so`` for sm_100a with nvcc.

Translation units with different numerics:
  flush.cu      -fmad=false: every float expression of the flush is rounded
                 exactly as written (bit-exact with the reference's CPU path);
  attention.cu, tree_attention.cu, shared_attention.cu  default contraction (FMA) for the attention math;
  reorder.cu    moves rows, no arithmetic;
  beam.cu       default contraction (its float64 scores decide);
  rotary.cu, logits.cu  default contraction;
  plugin.cu, unified.cu  -fmad=false: the operator-level plugin functions, same contract as flush.cu.
and ``host_file()``, the CPython binding of the calls whose time is the host's (host.cpp, g++).
Run ``python -m logkv_b200.build`` (or ``__graft_entry__.build()``).
"""
from __future__ import annotations

import os
import shutil
import subprocess
import sys
import sysconfig

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
CSRC = os.path.join(HERE, "csrc")
LIB = os.path.join(HERE, "liblogkv_b200.so")
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
COMMON = ["-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC", "-Xcompiler", "-fvisibility=hidden",
          f"-I{ROOT}", "--expt-relaxed-constexpr"]

UNITS = [
    ("flush.cu", ["-fmad=false"]),
    ("attention.cu", []),
    ("tree_attention.cu", []),
    ("shared_attention.cu", []),
    ("reorder.cu", []),
    ("beam.cu", []),
    ("rotary.cu", []),
    ("logits.cu", []),
    ("plugin.cu", ["-fmad=false"]),
    ("unified.cu", ["-fmad=false"]),
]


def nvcc() -> str:
    path = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(path):
        raise RuntimeError("nvcc not found; the CUDA toolkit is required to build logkv_b200")
    return path


def sources_newer_than(target: str, suffixes=(".cu", ".cuh")) -> bool:
    if not os.path.exists(target):
        return True
    t = os.path.getmtime(target)
    for root in (CSRC, os.path.join(ROOT, "include")):
        for name in os.listdir(root):
            if name.endswith((".h", *suffixes)) and os.path.getmtime(os.path.join(root, name)) > t:
                return True
    return False


def host_file() -> str:
    """The binding's path, with the torch version and the interpreter's ABI it is built against: either's
    C++ or C interface changes, so another one's file is neither loaded nor taken for built."""
    import torch
    return os.path.join(HERE, f"_host.torch{torch.__version__}{sysconfig.get_config_var('EXT_SUFFIX')}")


def build_host() -> None:
    """The CPython binding against this interpreter's torch."""
    import torch
    base = os.path.dirname(torch.__file__)
    inc = [os.path.join(base, "include"), os.path.join(base, "include", "torch", "csrc", "api", "include"),
           os.path.join(os.path.dirname(os.path.dirname(os.path.realpath(nvcc()))), "include")]
    tmp = host_file() + ".tmp"
    subprocess.run(["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden",
                    f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
                    "-I" + sysconfig.get_paths()["include"], *(x for i in inc for x in ("-isystem", i)),
                    os.path.join(CSRC, "host.cpp"), "-o", tmp, "-L" + os.path.join(base, "lib"), "-lc10", "-lc10_cuda",
                    "-ltorch_cpu", "-ltorch_python"], check=True)
    os.replace(tmp, host_file())


def build(force: bool = False, verbose: bool = False) -> str:
    if force or sources_newer_than(host_file(), (".cpp",)):
        build_host()
    if not force and not sources_newer_than(LIB):
        return LIB
    objdir = os.path.join(HERE, "_build")
    os.makedirs(objdir, exist_ok=True)
    objs, running = [], []
    for unit, extra in UNITS:   # the units compile side by side
        src = os.path.join(CSRC, unit)
        if not os.path.exists(src):
            continue
        obj = os.path.join(objdir, unit.replace(".cu", ".o"))
        cmd = [nvcc(), *ARCH, *COMMON, *extra, "-c", src, "-o", obj]
        if verbose:
            cmd.insert(1, "-Xptxas=-v")
            print(" ".join(cmd), flush=True)
        running.append((cmd, subprocess.Popen(cmd)))
        objs.append(obj)
    for cmd, p in running:
        if p.wait():
            for _, other in running:
                other.wait()
            raise subprocess.CalledProcessError(p.returncode, cmd)
    tmp = LIB + ".tmp"
    subprocess.run([nvcc(), *ARCH, "-shared", "-o", tmp, *objs, "-lcudart"], check=True)
    os.replace(tmp, LIB)
    return LIB


if __name__ == "__main__":
    build(force="--force" in sys.argv, verbose="-v" in sys.argv)
    print(LIB)
