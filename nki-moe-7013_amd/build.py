"""Build libqmoe.so (gfx950) in-tree from csrc/.

    python nki-moe-7013_amd/build.py [-j N]

Each csrc/*.hip / *.cpp is compiled by hipcc into _build/*.o (in parallel),
then linked into qmoe/libqmoe.so next to the Python bindings; bind/native.cpp
(host code against torch's headers) becomes the extension module
qmoe/_native.so, which links to it; probes/*.hip (measurement kernels that
bench.py uses for measured peaks, not part of the C ABI) go into
qmoe/libqmoe_probe.so.  Every HIP translation unit is built
with packed-FP32 instruction selection disabled.  The libraries need hipcc
alone: without torch the extension module, which only qmoe/ops.py loads, is
left out.
"""

from __future__ import annotations

import argparse
import concurrent.futures as cf
import json
import os
import shutil
import subprocess
import sys
import sysconfig

PKG = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(PKG)
CSRC = os.path.join(PKG, "csrc")
OUT_DIR = os.path.join(PKG, "_build")
LIB = os.path.join(PKG, "qmoe", "libqmoe.so")
NATIVE_SRC = os.path.join(PKG, "bind", "native.cpp")
NATIVE = os.path.join(PKG, "qmoe", "_native.so")
PROBES = os.path.join(PKG, "probes")
PROBE_LIB = os.path.join(PKG, "qmoe", "libqmoe_probe.so")
BUILD_INFO = os.path.join(PKG, "qmoe", "build_info.json")
ARCH = "gfx950"

COMMON = [
    "-O3",
    "-std=c++17",
    "-fPIC",
    f"--offload-arch={ARCH}",
    "-I" + os.path.join(ROOT, "include"),
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
    "-Wall",
    "-Wno-unused-function",
]


def hipcc() -> str:
    for cand in (os.environ.get("HIPCC"), "/opt/rocm/bin/hipcc", shutil.which("hipcc")):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("hipcc not found (ROCm is required to build libqmoe)")


def _compile(src: str) -> str:
    obj = os.path.join(OUT_DIR, os.path.basename(src) + ".o")
    cmd = [hipcc(), *COMMON, "-c", src, "-o", obj]
    r = subprocess.run(cmd, capture_output=True, text=True)
    msgs = "\n".join(
        l for l in (r.stdout + r.stderr).splitlines() if "packed-fp32-ops" not in l
    ).strip()
    if r.returncode != 0:
        raise RuntimeError(f"compile failed: {src}\n{msgs}")
    if msgs:
        print(msgs, file=sys.stderr)
    return obj


def _build_native() -> None:
    """The extension module, with the host compiler: no device code in it."""
    try:
        import torch
        from torch.utils import cpp_extension
    except ImportError as e:
        if os.path.exists(NATIVE):  # of an earlier library
            os.remove(NATIVE)
        print(f"qmoe/_native.so (the cache operators of qmoe/ops.py) is not built: {e}", file=sys.stderr)
        return
    lib_dir = os.path.join(os.path.dirname(torch.__file__), "lib")
    rocm = os.path.dirname(os.path.dirname(hipcc()))
    includes = [*cpp_extension.include_paths(), sysconfig.get_paths()["include"], os.path.join(rocm, "include"),
                os.path.join(ROOT, "include")]
    cxx = shutil.which("g++") or shutil.which("c++") or os.path.join(rocm, "llvm", "bin", "clang++")
    cmd = [cxx, "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden",
           "-D__HIP_PLATFORM_AMD__", "-DUSE_ROCM", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
           *[f"-I{i}" for i in includes], NATIVE_SRC, "-o", NATIVE + ".tmp", f"-L{lib_dir}", "-ltorch_python",
           "-ltorch_cpu", "-lc10", "-lc10_hip", f"-L{os.path.dirname(LIB)}", "-l:libqmoe.so", "-Wl,-rpath,$ORIGIN",
           f"-Wl,-rpath,{lib_dir}"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError("native module failed:\n" + r.stdout + r.stderr)
    os.replace(NATIVE + ".tmp", NATIVE)


def build(jobs: int = 8) -> str:
    os.makedirs(OUT_DIR, exist_ok=True)
    srcs = sorted(
        os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith((".hip", ".cpp"))
    )
    with cf.ThreadPoolExecutor(max_workers=max(1, jobs)) as ex:
        objs = list(ex.map(_compile, srcs))
    tmp = LIB + ".tmp"
    cmd = [hipcc(), f"--offload-arch={ARCH}", "-shared", "-fPIC", "-o", tmp, *objs, "-lhipblaslt"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError("link failed:\n" + r.stdout + r.stderr)
    os.replace(tmp, LIB)
    # measurement probes (bench.py's measured peaks): a library of their own
    psrcs = sorted(os.path.join(PROBES, f) for f in os.listdir(PROBES) if f.endswith(".hip"))
    pobjs = [_compile(p) for p in psrcs]
    cmd = [hipcc(), f"--offload-arch={ARCH}", "-shared", "-fPIC", "-o", PROBE_LIB + ".tmp", *pobjs]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError("probe link failed:\n" + r.stdout + r.stderr)
    os.replace(PROBE_LIB + ".tmp", PROBE_LIB)
    _write_build_info()
    _build_native()
    return LIB


def _write_build_info() -> None:
    """Record the commit the library was built from next to it (a copy of
    the tree without .git can still name its commit: bench.py reads this file)."""
    def git(*args):
        try:
            return subprocess.run(["git", *args], cwd=ROOT, capture_output=True, text=True,
                                  timeout=10).stdout.strip()
        except (OSError, subprocess.SubprocessError):
            return ""
    info = {"git": git("rev-parse", "--short", "HEAD") or None,
            "dirty": bool(git("status", "--porcelain", "--untracked-files=no"))}
    with open(BUILD_INFO, "w") as f:
        json.dump(info, f)


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("-j", "--jobs", type=int, default=min(8, os.cpu_count() or 1))
    a = ap.parse_args()
    print(build(a.jobs))
