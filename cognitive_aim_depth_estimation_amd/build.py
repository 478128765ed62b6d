"""Builds libcogaim.so (hipcc, gfx950 only) and the host module of training.py in-tree next to the sources."""
from __future__ import annotations

import os
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
LIB = os.path.join(HERE, "libcogaim.so")
HOST = os.path.join(HERE, "_host.so")            # host side of training.py: a Python module on torch's C++ API
SOURCES = ["gemm.hip", "gemm_rowln.hip", "attention.hip", "rowwise.hip", "focal.hip", "small.hip", "preprocess.hip",
           "train_rows.hip", "train_linear.hip"]
# attention.hip: without NaN-honouring, fmaxf on MFMA results needs no canonicalising v_max (x3 fewer max ops)
EXTRA_FLAGS = {"attention.hip": ["-fno-honor-nans"],
               "train_rows.hip": ["-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops"],     # no packed fp32 arithmetic
               "train_linear.hip": ["-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops"]}


def _hipcc() -> str:
    for cand in (os.environ.get("HIPCC"), "/opt/rocm/bin/hipcc", "hipcc"):
        if cand and (os.path.sep not in cand or os.path.exists(cand)):
            return cand
    raise RuntimeError("hipcc not found")


def needs_build() -> bool:
    if not os.path.exists(LIB) or not os.path.exists(HOST):
        return True
    t = min(os.path.getmtime(LIB), os.path.getmtime(HOST))
    deps = [os.path.join(CSRC, f) for f in os.listdir(CSRC)] + [os.path.join(HERE, "..", "include", "cogaim.h")]
    return any(os.path.getmtime(d) > t for d in deps)


def _host_command():
    import sysconfig

    import torch
    root = os.path.dirname(torch.__file__)
    return ["g++", "-O2", "-std=c++17", "-shared", "-fPIC", "-w", "-D__HIP_PLATFORM_AMD__=1", "-DUSE_ROCM=1", "-I" + os.path.join(root, "include"),
            "-I" + os.path.join(root, "include", "torch", "csrc", "api", "include"), "-I/opt/rocm/include",
            "-I" + sysconfig.get_paths()["include"], os.path.join(CSRC, "host_training.cpp"), "-o", HOST, "-L" + os.path.join(root, "lib"),
            "-ltorch_python", "-ltorch", "-ltorch_cpu", "-ltorch_hip", "-lc10", "-lc10_hip"]


def build(force: bool = False, verbose: bool = True) -> str:
    if not force and not needs_build():
        return LIB
    objs = []
    procs = []
    os.makedirs(os.path.join(HERE, "build"), exist_ok=True)
    for src in SOURCES:
        obj = os.path.join(HERE, "build", src.replace(".hip", ".o"))
        cmd = [_hipcc(), "--offload-arch=gfx950", "-O3", "-std=c++17", "-fPIC"] + EXTRA_FLAGS.get(src, []) + [
            "-c", os.path.join(CSRC, src), "-o", obj]
        if verbose:
            print(" ".join(cmd), flush=True)
        procs.append((src, subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT)))
        objs.append(obj)
    cmd = _host_command()
    if verbose:
        print(" ".join(cmd), flush=True)
    procs.append(("host_training.cpp", subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT)))
    for src, p in procs:
        out, _ = p.communicate()
        if p.returncode != 0:
            sys.stderr.write(out.decode())
            raise RuntimeError(f"the compiler failed on {src}")
    cmd = [_hipcc(), "--offload-arch=gfx950", "-shared", "-fPIC", "-o", LIB] + objs
    if verbose:
        print(" ".join(cmd), flush=True)
    subprocess.check_call(cmd)
    return LIB


if __name__ == "__main__":
    build(force="--force" in sys.argv)
    print(LIB)
