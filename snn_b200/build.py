"""Builds snn_b200/_lib/libsnn_b200.so (sm_100a) in-tree with nvcc.

    python -m snn_b200.build            # build if sources changed
    python -m snn_b200.build --force    # rebuild everything

cudart is linked statically (nvcc's default), so the library does not depend
on which libcudart the host process (e.g. PyTorch) already loaded. NCCL is the
one the installed PyTorch uses (the nvidia-nccl wheel), found through an
rpath, so a process that also runs torch.distributed loads a single NCCL.
snn_b200/_lib/sequence_ops.so, the sequence operators for torch tensors, is
built beside it with g++ against the installed PyTorch, and again when another
PyTorch or Python is found; without a CUDA build of PyTorch it is left out.
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
ROOT = os.path.dirname(HERE)
CSRC = os.path.join(HERE, "csrc")
OUT_DIR = os.path.join(HERE, "_lib")
OBJ_DIR = os.path.join(HERE, "_build")
LIB = os.path.join(OUT_DIR, "libsnn_b200.so")
TORCH_OPS = os.path.join(OUT_DIR, "sequence_ops.so")

ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
# --fmad=false: no FMA contraction anywhere (the reference's bit-parity rule,
# CMakeLists.txt:57-60); the kernels also use explicitly rounded intrinsics.
NVCC_FLAGS = ["-O3", "-lineinfo", "--fmad=false", "-std=c++17", "-Xcompiler", "-fPIC,-Wall",
              "--expt-relaxed-constexpr"]


def nvcc() -> str:
    for cand in (os.environ.get("NVCC"), "/usr/local/cuda/bin/nvcc", shutil.which("nvcc")):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found")


def nccl_dirs() -> tuple[str, str]:
    """Include and lib directory of the NCCL that PyTorch links."""
    cands = []
    for p in sys.path:
        cands.append(os.path.join(p, "nvidia", "nccl"))
    for d in cands:
        inc, lib = os.path.join(d, "include"), os.path.join(d, "lib")
        if os.path.exists(os.path.join(inc, "nccl.h")) and glob.glob(os.path.join(lib, "libnccl.so*")):
            return inc, lib
    if os.path.exists("/usr/include/nccl.h"):
        return "/usr/include", "/usr/lib/x86_64-linux-gnu"
    raise RuntimeError("nccl.h not found")


def _newer(src_files, target) -> bool:
    if not os.path.exists(target):
        return True
    t = os.path.getmtime(target)
    return any(os.path.getmtime(f) > t for f in src_files)


def torch_dir() -> str | None:
    """The installed PyTorch, if it has headers and was built for CUDA."""
    for p in sys.path:
        d = os.path.join(p, "torch")
        if os.path.exists(os.path.join(d, "include", "ATen", "ATen.h")):
            return d if os.path.exists(os.path.join(d, "lib", "libc10_cuda.so")) else None
    return None


def torch_stamp(t: str) -> str:
    """What the binary of the tensor operators depends on beside its sources."""
    with open(os.path.join(t, "version.py")) as f:
        return f"{sys.implementation.cache_tag} {t}\n{f.read()}"


def build_torch_ops(headers, force: bool, verbose: bool) -> None:
    t = torch_dir()
    if t is None:
        print(f"PyTorch for CUDA not found: {os.path.basename(TORCH_OPS)} (operators on torch tensors) not built",
              file=sys.stderr)
        return
    src = os.path.join(CSRC, "torch", "sequence_ops.cpp")
    stamp, now = os.path.join(OBJ_DIR, "sequence_ops.stamp"), torch_stamp(t)
    same = False
    if os.path.exists(stamp):
        with open(stamp) as f:
            same = f.read() == now
    if not (force or not same or _newer([src] + headers, TORCH_OPS)):
        return
    cuda = os.path.dirname(os.path.dirname(nvcc()))
    cmd = ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-Wall", "-I", os.path.join(ROOT, "include"),
           "-I", os.path.join(t, "include"), "-I", os.path.join(t, "include", "torch", "csrc", "api", "include"),
           "-I", os.path.join(cuda, "include"), "-I", sysconfig.get_paths()["include"], src, "-o", TORCH_OPS,
           "-L", os.path.join(t, "lib"), "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch_python",
           "-L", OUT_DIR, "-lsnn_b200", "-Wl,-rpath,$ORIGIN", "-Wl,-rpath," + os.path.join(t, "lib")]
    if verbose:
        print(" ".join(cmd))
    subprocess.run(cmd, check=True)
    with open(stamp, "w") as f:
        f.write(now)


def build(force: bool = False, verbose: bool = False) -> str:
    os.makedirs(OUT_DIR, exist_ok=True)
    os.makedirs(OBJ_DIR, exist_ok=True)
    srcs = sorted(glob.glob(os.path.join(CSRC, "*.cu")))
    headers = sorted(glob.glob(os.path.join(CSRC, "*.h")) + glob.glob(os.path.join(CSRC, "*.cuh")) +
                     glob.glob(os.path.join(ROOT, "include", "*.h")))
    inc, lib = nccl_dirs()
    cc = nvcc()
    incs = ["-I", os.path.join(ROOT, "include"), "-I", CSRC, "-I", inc]

    def compile_one(src):
        obj = os.path.join(OBJ_DIR, os.path.basename(src) + ".o")
        if force or _newer([src] + headers, obj):
            cmd = [cc, *ARCH, *NVCC_FLAGS, *incs, "-c", src, "-o", obj]
            if verbose:
                print(" ".join(cmd))
            subprocess.run(cmd, check=True)
        return obj

    with cf.ThreadPoolExecutor(max_workers=len(srcs)) as ex:
        objs = list(ex.map(compile_one, srcs))
    if force or _newer(objs, LIB):
        nccl_so = sorted(glob.glob(os.path.join(lib, "libnccl.so*")))[0]
        cmd = [cc, *ARCH, "-shared", "-Xcompiler", "-fPIC", "-o", LIB, *objs,
               "-L", lib, "-l:" + os.path.basename(nccl_so), "-Xlinker", "-rpath," + lib]
        if verbose:
            print(" ".join(cmd))
        subprocess.run(cmd, check=True)
    build_torch_ops([h for h in headers if h.startswith(os.path.join(ROOT, "include"))], force, verbose)
    return LIB


def main():
    ap = argparse.ArgumentParser()
    ap.add_argument("--force", action="store_true")
    ap.add_argument("-v", "--verbose", action="store_true")
    a = ap.parse_args()
    print(build(force=a.force, verbose=a.verbose))


if __name__ == "__main__":
    main()
