#!/usr/bin/env python
"""Build libatflash_b200.so (sm_100a) in-tree with nvcc, and the Python binding of its
short calls with g++ (against the installed torch's headers).

    python atflash-kernel_b200/build.py [--verbose-ptxas]

The library is written to atflash-kernel_b200/atflash/_lib/, the binding to
atflash-kernel_b200/atflash/_binding<suffix>, with the extension suffix of the Python that
runs this (no other Python loads it), so that they travel with the source tree; nothing is
installed. Beside the binding stands the version of torch that it was built against: with
another torch it is built again.
"""
import argparse
import importlib.util
import os
import re
import shutil
import subprocess
import sys
import sysconfig

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
CSRC = os.path.join(HERE, "csrc")
OUT_DIR = os.path.join(HERE, "atflash", "_lib")
LIB = os.path.join(OUT_DIR, "libatflash_b200.so")
BINDING = os.path.join(HERE, "atflash", "_binding" + sysconfig.get_config_var("EXT_SUFFIX"))
SOURCES = ["api.cu", "prefill_sm100.cu", "prefill_ragged_sm100.cu", "prefill_paged_sm100.cu", "decode.cu",
           "decode_e4m3.cu", "decode_noalloc.cu", "exchange.cu", "rope.cu", "append.cu", "append_e4m3.cu", "tables.cu", "pages.cu", "qk_norm.cu",
           "selftest.cu"]
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]


def nvcc_path():
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found")


def build_library(verbose_ptxas=False, force=False):
    os.makedirs(OUT_DIR, exist_ok=True)
    srcs = [os.path.join(CSRC, s) for s in SOURCES]
    deps = srcs + [os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith((".cuh", ".h"))]
    deps.append(os.path.join(ROOT, "include", "atflash_b200.h"))
    if not force and os.path.exists(LIB):
        t = os.path.getmtime(LIB)
        if all(os.path.getmtime(d) <= t for d in deps):
            return LIB
    cmd = [nvcc_path(), "-O3", "-std=c++17", *ARCH, "-lineinfo", "-Xcompiler", "-fPIC",
           "-shared", "-I", os.path.join(ROOT, "include"), "-o", LIB + ".tmp", *srcs]
    if verbose_ptxas:
        cmd[1:1] = ["-Xptxas", "-v"]
    subprocess.run(cmd, check=True)
    os.replace(LIB + ".tmp", LIB)
    return LIB


def torch_version(torch_dir):
    """torch.__version__, without the import"""
    with open(os.path.join(torch_dir, "version.py")) as f:
        return re.search(r"^__version__\s*=\s*['\"]([^'\"]+)", f.read(), re.M).group(1)


def build_binding(force=False):
    src = os.path.join(CSRC, "binding.cpp")
    torch_dir = os.path.dirname(importlib.util.find_spec("torch").origin)
    # file times say nothing of the installed torch, which may be older than the binding
    stamp, version = BINDING + ".torch", torch_version(torch_dir)
    deps = [src, os.path.join(ROOT, "include", "atflash_b200.h")]
    if not force and os.path.exists(BINDING) and os.path.exists(stamp):
        t = os.path.getmtime(BINDING)
        with open(stamp) as f:
            built_for = f.read()
        if built_for == version and all(os.path.getmtime(d) <= t for d in deps):
            return BINDING
    cuda = os.path.dirname(os.path.dirname(os.path.realpath(nvcc_path())))
    inc = [os.path.join(torch_dir, "include"), os.path.join(torch_dir, "include", "torch", "csrc", "api", "include"),
           sysconfig.get_paths()["include"], os.path.join(cuda, "include")]
    cmd = [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-fPIC", "-shared", *(f"-I{i}" for i in inc), "-o",
           BINDING + ".tmp", src, f"-L{os.path.join(torch_dir, 'lib')}",
           *(f"-l{lib}" for lib in ("c10", "c10_cuda", "torch_cpu", "torch", "torch_python"))]
    subprocess.run(cmd, check=True)
    if os.path.exists(stamp):
        os.remove(stamp)
    os.replace(BINDING + ".tmp", BINDING)
    with open(stamp, "w") as f:
        f.write(version)
    untagged = os.path.join(os.path.dirname(BINDING), "_binding.so")
    if os.path.exists(untagged):  # of an earlier build: any Python would load it
        os.remove(untagged)
    return BINDING


def build(verbose_ptxas=False, force=False):
    lib = build_library(verbose_ptxas, force)
    build_binding(force)
    return lib


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--verbose-ptxas", action="store_true")
    ap.add_argument("--force", action="store_true")
    a = ap.parse_args()
    print(build(a.verbose_ptxas, a.force))
    sys.exit(0)
