"""Build the sm_100a CUDA library in-tree: strands_decider_b200/lib/libstrands_b200.so.

    python -m strands_decider_b200.build [--force] [-j N]

Each .cu in csrc/ is compiled for sm_100a only (`-gencode arch=compute_100a,code=sm_100a`)
as relocatable device code, then device-linked into one shared library. Rebuilds only
when a source or header is newer than the library (or with --force).

csrc/int8_torch.cpp becomes the Python extension module _int8_ops, in the same folder: host code over
torch's headers, which takes the library's entry points by address and links nothing of it. It is
compiled against one torch and one Python, so its file is named after both: after a change of either
it is missing, not loaded against other layouts. Processes that build at once take turns.
"""

from __future__ import annotations

import argparse
import contextlib
import fcntl
import glob
import os
import re
import shutil
import subprocess
import sys
import sysconfig
from concurrent.futures import ThreadPoolExecutor

PKG = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(PKG)
CSRC = os.path.join(PKG, "csrc")
INCLUDE = os.path.join(ROOT, "include")
LIBDIR = os.path.join(PKG, "lib")
LIB = os.path.join(LIBDIR, "libstrands_b200.so")
OBJDIR = os.path.join(PKG, "_build")
OPS_SRC = os.path.join(CSRC, "int8_torch.cpp")

ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
FLAGS = ["-O3", "-lineinfo", "-std=c++17", "-rdc=true", "-Xcompiler", "-fPIC,-O2", "--expt-relaxed-constexpr",
         "-Xptxas", "-warn-spills", f"-I{INCLUDE}", f"-I{CSRC}"]


def nvcc() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found; the B200 library needs the CUDA 12.9 toolkit")


def sources() -> list[str]:
    return sorted(glob.glob(os.path.join(CSRC, "*.cu")))


def _inputs() -> list[str]:
    return sources() + glob.glob(os.path.join(CSRC, "*.cuh")) + glob.glob(os.path.join(INCLUDE, "*.h")) + [__file__]


def up_to_date() -> bool:
    if not os.path.exists(LIB):
        return False
    t = os.path.getmtime(LIB)
    return all(os.path.getmtime(p) <= t for p in _inputs())


@contextlib.contextmanager
def _turn():
    """One build at a time in this tree."""
    os.makedirs(LIBDIR, exist_ok=True)
    os.makedirs(OBJDIR, exist_ok=True)
    with open(os.path.join(OBJDIR, "lock"), "w") as f:
        fcntl.flock(f, fcntl.LOCK_EX)
        yield


def ops_path() -> str:
    """The extension module of the int8 operators' Python calls, for the running torch and Python."""
    import torch

    abi = "" if torch.compiled_with_cxx11_abi() else "-precxx11"
    version = re.sub(r"[^\w.]", "_", f"{torch.__version__}-{(torch.version.git_version or '')[:10]}")
    return os.path.join(LIBDIR, f"_int8_ops-torch{version}{abi}{sysconfig.get_config_var('EXT_SUFFIX')}")


def ops_up_to_date() -> bool:
    ops = ops_path()
    inputs = [OPS_SRC, os.path.join(INCLUDE, "strands_b200.h"), __file__]
    return os.path.exists(ops) and all(os.path.getmtime(p) <= os.path.getmtime(ops) for p in inputs)


def _compile_ops() -> None:
    import torch

    root = os.path.dirname(torch.__file__)
    ops = ops_path()
    tmp = f"{ops}.{os.getpid()}.tmp"
    cmd = [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-shared", "-fPIC",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch.compiled_with_cxx11_abi())}", f"-I{INCLUDE}",
           "-isystem", sysconfig.get_paths()["include"], "-isystem", os.path.join(root, "include"),
           "-isystem", os.path.join(root, "include", "torch", "csrc", "api", "include"),
           OPS_SRC, "-o", tmp, "-L" + os.path.join(root, "lib"), "-ltorch_python", "-ltorch_cpu", "-lc10"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"{cmd[0]} failed on {os.path.basename(OPS_SRC)}:\n{r.stdout}\n{r.stderr}")
    os.replace(tmp, ops)


def build_ops(force: bool = False) -> str:
    """Build the extension module where it is missing or older than its sources."""
    if force or not ops_up_to_date():
        with _turn():
            if force or not ops_up_to_date():   # another process may have built it meanwhile
                _compile_ops()
    return ops_path()


def build(force: bool = False, jobs: int | None = None, verbose: bool = False, extra: list[str] | None = None) -> str:
    build_ops(force)
    if force or not up_to_date():
        with _turn():
            if force or not up_to_date():
                _compile_library(jobs, verbose, extra or [])
    return LIB


def _compile_library(jobs: int | None, verbose: bool, extra: list[str]) -> None:
    cc = nvcc()

    def compile_one(src: str) -> str:
        obj = os.path.join(OBJDIR, os.path.basename(src)[:-3] + ".o")
        cmd = [cc, *ARCH, *FLAGS, *extra, "-c", src, "-o", obj]
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"nvcc failed on {os.path.basename(src)}:\n{r.stdout}\n{r.stderr}")
        if verbose and (r.stdout or r.stderr):
            print(r.stdout + r.stderr, file=sys.stderr)
        return obj

    with ThreadPoolExecutor(max_workers=jobs or os.cpu_count() or 4) as ex:
        objs = list(ex.map(compile_one, sources()))
    tmp = f"{LIB}.{os.getpid()}.tmp"
    cmd = [cc, *ARCH, "-shared", "-Xcompiler", "-fPIC", "-o", tmp, *objs, "-lcudart_static", "-ldl", "-lrt", "-lpthread"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"link failed:\n{r.stdout}\n{r.stderr}")
    os.replace(tmp, LIB)


def main() -> None:
    ap = argparse.ArgumentParser()
    ap.add_argument("--force", action="store_true")
    ap.add_argument("-j", type=int, default=None)
    ap.add_argument("-v", action="store_true")
    ap.add_argument("--ptxas-v", action="store_true", help="print registers / spills per kernel")
    a = ap.parse_args()
    extra = ["-Xptxas", "-v"] if a.ptxas_v else None
    print(build(force=a.force or a.ptxas_v, jobs=a.j, verbose=a.v or a.ptxas_v, extra=extra))


if __name__ == "__main__":
    main()
