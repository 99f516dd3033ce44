"""Build ``wisp_b200/lib/libwisp_b200.so`` from ``wisp_b200/csrc`` with nvcc, and the Python binding of the stateless
operators (``wisp_b200/lib/_wisp_bind.so``, ``csrc/bind.cpp`` against torch's headers) with g++.

sm_100a only (B200).  The library links the CUDA runtime statically and
reaches no driver symbol at load time, so it also loads (for symbol checks)
on a machine without a GPU.

    python -m wisp_b200.build          # incremental
    python -m wisp_b200.build --force
"""
from __future__ import annotations

import argparse
import glob
import importlib.metadata
import os
import shutil
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
LIBDIR = os.path.join(HERE, "lib")
LIB = os.path.join(LIBDIR, "libwisp_b200.so")
BIND_SRC = os.path.join(CSRC, "bind.cpp")
BIND = os.path.join(LIBDIR, "_wisp_bind.so")
BIND_STAMP = os.path.join(LIBDIR, "_wisp_bind.stamp")
INCLUDE = os.path.join(os.path.dirname(HERE), "include")

ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
FLAGS = ["-O3", "-std=c++17", "-lineinfo", "--expt-relaxed-constexpr",
         "-Xcompiler", "-fPIC", "-Xcompiler", "-fvisibility=hidden",
         "-Xcompiler", "-Wall", "-diag-suppress", "177"]


def _nvcc() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found: the CUDA toolkit is required to build wisp_b200")


def sources() -> list[str]:
    return sorted(glob.glob(os.path.join(CSRC, "*.cu")))


def _stale() -> bool:
    if not os.path.exists(LIB):
        return True
    t = os.path.getmtime(LIB)
    deps = sources() + glob.glob(os.path.join(CSRC, "*.cuh")) + glob.glob(os.path.join(INCLUDE, "*.h"))
    return any(os.path.getmtime(d) > t for d in deps)


def _bind_made_for() -> str:
    """What the binding depends on besides its sources: the interpreter's and torch's binary interfaces."""
    try:
        torch_version = importlib.metadata.version("torch")
    except importlib.metadata.PackageNotFoundError:
        torch_version = "none"
    return f"{sys.implementation.cache_tag} torch {torch_version}"


def build_bind(force: bool = False) -> str | None:
    """The Python binding; it finds ``libwisp_b200.so`` beside itself.  Rebuilt when its sources, the interpreter or
    torch's version changed.  Without torch there is nothing to build it against, and nothing to use it with: None."""
    header = os.path.join(INCLUDE, "wisp_b200.h")
    made_for = _bind_made_for()
    if not force and os.path.exists(BIND) and all(os.path.getmtime(p) <= os.path.getmtime(BIND)
                                                  for p in (BIND_SRC, header)):
        if os.path.exists(BIND_STAMP) and open(BIND_STAMP).read() == made_for:
            return BIND
    try:
        import torch
    except ImportError:
        print("wisp_b200: no torch, so the Python binding of the stateless operators is not built", file=sys.stderr)
        return None
    import sysconfig
    tree = os.path.dirname(torch.__file__)
    cuda = os.path.dirname(os.path.dirname(_nvcc()))
    inc = [os.path.join(tree, "include"), os.path.join(tree, "include", "torch", "csrc", "api", "include"),
           os.path.join(cuda, "include"), sysconfig.get_paths()["include"]]
    tmp = BIND + ".tmp"
    cmd = ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", *[f"-I{p}" for p in inc], BIND_SRC,
           "-o", tmp, f"-L{LIBDIR}", "-lwisp_b200", "-Wl,-rpath,$ORIGIN", f"-L{os.path.join(tree, 'lib')}", "-lc10",
           "-lc10_cuda", "-ltorch_cpu", "-ltorch", "-ltorch_python"]
    subprocess.run(cmd, check=True)
    os.replace(tmp, BIND)
    with open(BIND_STAMP, "w") as f:
        f.write(made_for)
    return BIND


def build(force: bool = False, verbose: bool = False) -> str:
    if not force and not _stale():
        build_bind()
        return LIB
    os.makedirs(LIBDIR, exist_ok=True)
    objdir = os.path.join(LIBDIR, "_obj")
    os.makedirs(objdir, exist_ok=True)
    nvcc = _nvcc()
    cmds, objs = [], []
    for src in sources():
        obj = os.path.join(objdir, os.path.basename(src).replace(".cu", ".o"))
        cmd = [nvcc, *ARCH, *FLAGS, "-I", INCLUDE, "-c", src, "-o", obj]
        if verbose:
            cmd.insert(1, "-Xptxas=-v")
            print(" ".join(cmd), flush=True)
        cmds.append(cmd)
        objs.append(obj)
    # one nvcc per translation unit, in parallel
    with ThreadPoolExecutor(max_workers=max(1, min(len(cmds), os.cpu_count() or 1))) as pool:
        for r in pool.map(lambda c: subprocess.run(c, capture_output=not verbose, text=True), cmds):
            if r.returncode:
                sys.stderr.write((r.stdout or "") + (r.stderr or ""))
                raise subprocess.CalledProcessError(r.returncode, r.args)
    tmp = LIB + ".tmp"
    subprocess.run([nvcc, *ARCH, "-shared", "-cudart", "static", "-o", tmp, *objs], check=True)
    os.replace(tmp, LIB)
    build_bind(force)
    return LIB


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--force", action="store_true")
    ap.add_argument("-v", "--verbose", action="store_true")
    args = ap.parse_args()
    print(build(force=args.force, verbose=args.verbose))
    sys.exit(0)
