"""Build libspx.so (the C-ABI CUDA library) in-tree for sm_100a, and _spx_front.so (its
tensor-level entry points for the calls of a decode step, spx_front.cpp, against the torch of
this interpreter).

    python unsloth-spectral_b200/csrc/build.py [--jobs N] [--force]

Objects go to ``csrc/_build/``; the shared library is written next to the Python
package (``unsloth_spectral/libspx.so``) so it travels with the source tree.
"""
from __future__ import annotations

import argparse
import concurrent.futures as cf
import glob
import os
import shutil
import subprocess
import sys

CSRC = os.path.dirname(os.path.abspath(__file__))
PKG_ROOT = os.path.dirname(CSRC)
REPO = os.path.dirname(PKG_ROOT)
INCLUDE = os.path.join(REPO, "include")
OUT = os.path.join(PKG_ROOT, "unsloth_spectral", "libspx.so")
FRONT = os.path.join(PKG_ROOT, "unsloth_spectral", "_spx_front.so")
BUILD = os.path.join(CSRC, "_build")

ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
FLAGS = ["-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC", "-Xcompiler", "-fvisibility=hidden",
         "--expt-relaxed-constexpr", "-I", INCLUDE, "-I", CSRC]


def nvcc() -> str:
    for cand in (os.environ.get("NVCC"), "/usr/local/cuda/bin/nvcc", shutil.which("nvcc")):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found")


def _stale(obj: str, deps) -> bool:
    if not os.path.exists(obj):
        return True
    t = os.path.getmtime(obj)
    return any(os.path.getmtime(d) > t for d in deps)


def build(jobs: int = 0, force: bool = False, verbose: bool = False, ptxas_verbose: bool = False) -> str:
    os.makedirs(BUILD, exist_ok=True)
    sources = sorted(glob.glob(os.path.join(CSRC, "*.cu")))
    headers = glob.glob(os.path.join(CSRC, "*.cuh")) + glob.glob(os.path.join(INCLUDE, "*.h"))
    cc = nvcc()
    cmds = []
    objs = []
    for src in sources:
        obj = os.path.join(BUILD, os.path.basename(src)[:-3] + ".o")
        objs.append(obj)
        if force or _stale(obj, [src] + headers):
            extra = ["-Xptxas", "-v"] if ptxas_verbose else []
            cmds.append([cc, *ARCH, *FLAGS, *extra, "-c", src, "-o", obj])
    jobs = jobs or min(len(cmds) or 1, os.cpu_count() or 4)

    def run(cmd):
        r = subprocess.run(cmd, capture_output=True, text=True)
        return cmd, r

    failed = []
    with cf.ThreadPoolExecutor(max_workers=jobs) as ex:
        for cmd, r in ex.map(run, cmds):
            if verbose or r.returncode != 0 or ptxas_verbose:
                sys.stderr.write(r.stdout + r.stderr)
            if r.returncode != 0:
                failed.append(cmd[-3])
    if failed:
        raise RuntimeError(f"nvcc failed for: {failed}")
    if cmds or not os.path.exists(OUT) or force:
        link = [cc, *ARCH, "-shared", "-Xcompiler", "-fPIC", *objs, "-o", OUT]
        r = subprocess.run(link, capture_output=True, text=True)
        if r.returncode != 0:
            sys.stderr.write(r.stdout + r.stderr)
            raise RuntimeError("link failed")
    build_front(force)
    return OUT


def build_front(force: bool = False) -> str:
    import sysconfig

    import torch
    src = os.path.join(CSRC, "spx_front.cpp")
    # what it was built against, kept beside the objects: another torch or Python cannot load it
    record = os.path.join(BUILD, "front.txt")
    against = (f"torch {torch.__version__}, C++11 ABI {int(torch.compiled_with_cxx11_abi())}, "
               f"python {sysconfig.get_config_var('SOABI')}")
    if not force and not _stale(FRONT, [src, os.path.join(INCLUDE, "spx.h"), os.path.abspath(__file__)]):
        if os.path.exists(record) and open(record).read() == against:
            return FRONT
    root = os.path.dirname(torch.__file__)
    cuda = os.path.dirname(os.path.dirname(nvcc()))
    inc = [INCLUDE, os.path.join(root, "include"), os.path.join(root, "include", "torch", "csrc", "api", "include"),
           os.path.join(cuda, "include"), sysconfig.get_paths()["include"]]
    libs = ["c10", "c10_cuda", "torch_cpu", "torch_cuda", "torch", "torch_python"]
    cmd = ["g++", "-O2", "-std=c++17", "-fPIC", "-fvisibility=hidden", "-shared", "-DTORCH_API_INCLUDE_EXTENSION_H",
           "-DTORCH_EXTENSION_NAME=_spx_front", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch.compiled_with_cxx11_abi())}",
           *[f"-I{i}" for i in inc], src, "-o", FRONT, f"-L{os.path.join(root, 'lib')}", *[f"-l{n}" for n in libs],
           f"-L{os.path.dirname(OUT)}", "-lspx", "-Wl,-rpath,$ORIGIN"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        sys.stderr.write(r.stdout + r.stderr)
        raise RuntimeError("g++ failed for spx_front.cpp")
    os.makedirs(BUILD, exist_ok=True)
    with open(record, "w") as f:
        f.write(against)
    return FRONT


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--jobs", type=int, default=0)
    ap.add_argument("--force", action="store_true")
    ap.add_argument("--verbose", action="store_true")
    ap.add_argument("--ptxas", action="store_true", help="print -Xptxas -v register/smem usage")
    a = ap.parse_args()
    print(build(a.jobs, a.force, a.verbose, a.ptxas))
