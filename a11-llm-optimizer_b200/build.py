"""Build liba11spec.so (the C-ABI CUDA library) for sm_100a, in-tree.

Usage: python a11-llm-optimizer_b200/build.py [--force] [--verbose]
The library lands next to the Python package (a11spec/liba11spec.so) so that
it travels with the repository snapshot and is what the package loads.
"""
from __future__ import annotations

import argparse
import contextlib
import fcntl
import glob
import os
import subprocess
import sys
import tempfile

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
INCLUDE = os.path.join(os.path.dirname(HERE), "include")
OUT = os.path.join(HERE, "a11spec", "liba11spec.so")
CPP = os.path.join(HERE, "cpp")
FAST_DIR = os.path.join(HERE, "a11spec")
FAST_SOURCES = (os.path.join(CPP, "fast_ops.cpp"), os.path.join(INCLUDE, "a11spec.h"))
VERIFIER_OUT = os.path.join(CPP, "libspec_verifier.so")
CUDA_HOME = os.environ.get("CUDA_HOME", "/usr/local/cuda")
NVCC = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-O3", "-lineinfo", "-std=c++17",
    "-Xcompiler", "-fPIC", "-shared",
    "--expt-relaxed-constexpr",
    "-Xptxas", "-warn-spills",
]


@contextlib.contextmanager
def building(folder: str):
    """One process at a time builds into `folder`: under a lock on it (which leaves no
    file behind), with a scratch folder from which the result moves to its place whole."""
    lock = os.open(folder, os.O_RDONLY)
    try:
        with contextlib.suppress(OSError):  # no such locks there: several build, each in a folder of its own
            fcntl.flock(lock, fcntl.LOCK_EX)
        with tempfile.TemporaryDirectory(prefix=".build-", dir=folder) as tmp:
            yield tmp
    finally:
        os.close(lock)


def sources():
    return sorted(glob.glob(os.path.join(CSRC, "*.cu")))


def deps():
    return sources() + sorted(glob.glob(os.path.join(CSRC, "*.h")) + glob.glob(os.path.join(CSRC, "*.cuh"))) + [
        os.path.join(INCLUDE, "a11spec.h")]


def up_to_date() -> bool:
    if not os.path.exists(OUT):
        return False
    t = os.path.getmtime(OUT)
    return all(os.path.getmtime(p) <= t for p in deps())


def build(force: bool = False, verbose: bool = False, extra=()) -> str:
    if not force and up_to_date():
        return OUT
    with building(os.path.dirname(OUT)) as tmp:
        if not force and up_to_date():  # built by the one that held the lock
            return OUT
        made = os.path.join(tmp, "liba11spec.so")
        cmd = [NVCC, *NVCC_FLAGS, *extra, "-I", INCLUDE, "-o", made, *sources()]
        if verbose:
            cmd.insert(1, "-Xptxas=-v")
            print(" ".join(cmd), file=sys.stderr)
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError("nvcc failed:\n" + r.stdout + r.stderr)
        if verbose:
            print(r.stdout + r.stderr, file=sys.stderr)
        os.replace(made, OUT)
    return OUT


def build_verifier(force: bool = False) -> str:
    """libspec_verifier.so: the A11::Engine::SpeculativeTreeVerifier C++ interface
    over liba11spec (g++, links liba11spec.so and the CUDA runtime)."""
    src = os.path.join(CPP, "speculative_verifier.cpp")
    hdr = os.path.join(CPP, "include", "engine", "speculative_verifier.hpp")
    if not force and os.path.exists(VERIFIER_OUT) and all(
            os.path.getmtime(p) <= os.path.getmtime(VERIFIER_OUT) for p in (src, hdr, OUT)):
        return VERIFIER_OUT
    cmd = ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-I", os.path.join(CPP, "include"), "-I", INCLUDE,
           "-I", os.path.join(CUDA_HOME, "include"), "-o", VERIFIER_OUT, src, "-L", os.path.dirname(OUT),
           "-la11spec", "-Wl,-rpath,$ORIGIN/../a11spec", "-L", os.path.join(CUDA_HOME, "lib64"), "-lcudart"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError("g++ failed:\n" + r.stdout + r.stderr)
    return VERIFIER_OUT


def fast_path() -> str:
    """Where this interpreter's and this torch's a11spec._fast belongs: the name carries
    what it is compiled against and its sources, so that no other build is taken for it."""
    import hashlib
    import sysconfig

    import torch
    abi = "|".join((sysconfig.get_config_var("SOABI") or sys.version, torch.__version__, str(getattr(torch.version, "git_version", None)),
                    str(torch._C._GLIBCXX_USE_CXX11_ABI)))
    src = hashlib.sha256()
    for p in FAST_SOURCES:
        with open(p, "rb") as f:
            src.update(f.read())
    return os.path.join(FAST_DIR, f"_fast-{hashlib.sha256(abi.encode()).hexdigest()[:10]}-{src.hexdigest()[:10]}.so")


def build_fast(force: bool = False) -> str:
    """a11spec/_fast-*.so: the layer operators' argument checks and calls in C++
    (g++ against this interpreter's and this torch's headers). Safe to call from
    several processes at once: one builds, and the file appears when it is whole."""
    out = fast_path()
    if not force and os.path.exists(out):
        return out
    import sysconfig

    import torch
    root = os.path.dirname(torch.__file__)
    lib = os.path.join(root, "lib")
    inc = [INCLUDE, os.path.join(root, "include"), os.path.join(root, "include", "torch", "csrc", "api", "include"),
           os.path.join(CUDA_HOME, "include"), sysconfig.get_paths()["include"]]
    cmd = ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}"]
    for d in inc:
        cmd += ["-isystem" if d != INCLUDE else "-I", d]
    with building(FAST_DIR) as tmp:
        if not force and os.path.exists(out):  # built by the one that held the lock
            return out
        made = os.path.join(tmp, "_fast.so")
        r = subprocess.run(cmd + ["-o", made, FAST_SOURCES[0], "-L", os.path.dirname(OUT), "-la11spec", "-Wl,-rpath,$ORIGIN",
                                  "-L", lib, "-ltorch_python", "-ltorch", "-ltorch_cpu", "-lc10", "-lc10_cuda",
                                  f"-Wl,-rpath,{lib}"], capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError("g++ failed:\n" + r.stdout + r.stderr)
        os.replace(made, out)
        same_abi = out[:-len("-0123456789.so")]
        for old in glob.glob(glob.escape(same_abi) + "-*.so"):  # of earlier sources
            if old != out:
                with contextlib.suppress(FileNotFoundError):
                    os.remove(old)
    return out


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--force", action="store_true")
    ap.add_argument("--verbose", action="store_true")
    args = ap.parse_args()
    print(build(force=args.force, verbose=args.verbose))
    print(build_verifier(force=args.force))
    print(build_fast(force=args.force))
