"""Compile one group of HIP sources of ``csrc/`` into its shared library next to this file.

The package's kernels come in groups that build and load independently, so that a process pays only for what its model uses:
``pc_*.hip`` -> ``libpromptcache_hip.so`` (the split-precision fp16 stacks of the Llama / Falcon / MPT adapters) and
``pb_*.hip`` -> ``libpromptcache_blocks.so`` (the bf16 / fp32 building blocks), with it ``py_tensors.cpp`` -> ``_tensors.so`` (host code).  One hipcc per
translation unit, all at once.
"""
from __future__ import annotations

import contextlib
import fcntl
import glob
import os
import subprocess
import sys

PKG = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(os.path.dirname(PKG), "csrc")
INCLUDE = os.path.join(os.path.dirname(os.path.dirname(PKG)), "include")

GROUPS = {
    # group -> (source glob, library, extra flags)
    "blocks": ("pb_*.hip", "libpromptcache_blocks.so",
               # no packed-fp32 instructions: hipcc forms them from scalar float code by itself
               ["-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops"]),
}


def hipcc() -> str:
    for c in (os.environ.get("HIPCC"), "/opt/rocm/bin/hipcc", "hipcc"):
        if c and (os.path.isabs(c) and os.path.exists(c) or not os.path.isabs(c)):
            return c
    return "hipcc"


def lib_path(group: str) -> str:
    return os.path.join(PKG, GROUPS[group][1])


def stale(group: str) -> bool:
    pattern, _, _ = GROUPS[group]
    lib = lib_path(group)
    if not os.path.exists(lib):
        return True
    prefix = pattern.split("*")[0]
    deps = glob.glob(os.path.join(CSRC, pattern)) + glob.glob(os.path.join(CSRC, prefix + "*.h")) + \
        glob.glob(os.path.join(CSRC, "mfma_*.h")) + glob.glob(os.path.join(INCLUDE, "*.h"))
    return any(os.path.getmtime(d) > os.path.getmtime(lib) for d in deps)


def tensors_path() -> str:
    return os.path.join(PKG, "_tensors.so")


def tensors_stale() -> bool:
    """Whether ``_tensors.so`` is missing or older than its source.  (Whether it is this torch's: whoever loads it sees.)"""
    lib = tensors_path()
    return not os.path.exists(lib) or os.path.getmtime(os.path.join(CSRC, "py_tensors.cpp")) > os.path.getmtime(lib)


@contextlib.contextmanager
def _locked(group: str):
    """Concurrent builders of a group, one after the other."""
    objdir = os.path.join(CSRC, "_build")
    os.makedirs(objdir, exist_ok=True)
    with open(os.path.join(objdir, f".{group}.lock"), "w") as lock:
        fcntl.flock(lock, fcntl.LOCK_EX)
        yield objdir


def renew_tensors() -> None:
    """``_tensors.so`` anew, unless somebody else has just made it."""
    def made():
        return os.stat(tensors_path()).st_mtime_ns if os.path.exists(tensors_path()) else None
    seen = made()
    with _locked("blocks"):
        if made() == seen:
            build_tensors()


def build_tensors() -> None:
    """``py_tensors.cpp`` -> ``_tensors.so``, host code beside the blocks library.  Where Python's or torch's headers are missing it is left out: the wrappers then look at their
    tensors in Python."""
    import sysconfig

    import torch
    root = os.path.dirname(torch.__file__)
    lib = tensors_path()
    tmp = lib + f".{os.getpid()}.tmp"
    cmd = ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
           *(f"-I{d}" for d in (os.path.join(root, "include"), os.path.join(root, "include/torch/csrc/api/include"), sysconfig.get_paths()["include"])),
           os.path.join(CSRC, "py_tensors.cpp"), "-o", tmp, f"-L{os.path.join(root, 'lib')}", "-ltorch_python", "-ltorch_cpu", "-lc10"]
    print("[build]", " ".join(cmd), file=sys.stderr, flush=True)
    try:
        subprocess.check_call(cmd, stdout=sys.stderr)
    except (OSError, subprocess.CalledProcessError) as e:
        print(f"[build] without _tensors.so: {e}", file=sys.stderr, flush=True)
        return
    os.replace(tmp, lib)


def build(group: str, force: bool = False) -> str:
    """Build the group's library when it is missing or older than its sources (always with ``force``); returns its path.
    Concurrent callers serialise on a lock file, and the library appears under its name only when it is complete."""
    pattern, _, extra = GROUPS[group]
    lib = lib_path(group)
    with _locked(group) as objdir:
        if group == "blocks" and (force or tensors_stale()):
            build_tensors()
        if not force and not stale(group):
            return lib
        srcs = sorted(glob.glob(os.path.join(CSRC, pattern)))
        if not srcs:
            raise RuntimeError(f"no sources match {pattern} under {CSRC}")
        flags = ["--offload-arch=gfx950", "-O3", "-std=c++17", "-fPIC", "-fvisibility=hidden", *extra,
                 *os.environ.get("PC_BUILD_FLAGS", "").split()]
        jobs = []
        for src in srcs:
            obj = os.path.join(objdir, os.path.basename(src) + ".o")
            # (pb_linear_tiles.hip: up to 256 accumulator registers beside the operands, which only fit as AGPRs)
            form = [] if os.path.basename(src) == "pb_linear_tiles.hip" else ["-mllvm", "-amdgpu-mfma-vgpr-form"]
            cmd = [hipcc(), *flags, *form, "-c", src, "-o", obj]
            print("[build]", " ".join(cmd), file=sys.stderr, flush=True)
            jobs.append((obj, cmd, subprocess.Popen(cmd, cwd=os.path.dirname(CSRC), stdout=sys.stderr)))
        for obj, cmd, proc in jobs:
            if proc.wait() != 0:
                raise subprocess.CalledProcessError(proc.returncode, cmd)
        tmp = lib + f".{os.getpid()}.tmp"
        link = [hipcc(), "--offload-arch=gfx950", "-shared", "-fPIC", *[o for o, _, _ in jobs], "-o", tmp]
        print("[build]", " ".join(link), file=sys.stderr, flush=True)
        subprocess.check_call(link, cwd=os.path.dirname(CSRC), stdout=sys.stderr)
        os.replace(tmp, lib)
    return lib
