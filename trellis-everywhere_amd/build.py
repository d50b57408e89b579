"""Build the gfx950 HIP library libtrellis_amd.so in-tree with hipcc, and _serve.so, its binding for torch, with g++.

Run as ``python trellis-everywhere_amd/build.py`` or through ``__graft_entry__.build()``.
The .so lands next to this file so it travels with the source tree to the GPU box.
"""
from __future__ import annotations

import os
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
CSRC = os.path.join(HERE, "csrc")
LIB = os.path.join(HERE, "libtrellis_amd.so")
SOURCES = ["trellis_amd.hip", "kernels_k2.hip", "kernels_k3.hip", "kernels_k4.hip", "serve.hip"]
HEADERS = ["decode.h", "common.h", "gemv.h", "bgemm.h", "launch.h", "embed.h", "encode.h",
           "serve.h", "norm.h", "append.h", "attend_plan.h", "attend.h", "evict.h"]

# the Python side of the operators between the packed linears (host code against torch's C++ headers)
BIND = "bind.cpp"
BIND_LIB = os.path.join(HERE, "_serve.so")

HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
ARCH = "gfx950"
FLAGS = [
    f"--offload-arch={ARCH}",
    "-O3",
    "-std=c++17",
    "-fPIC",
    "-fhip-fp32-correctly-rounded-divide-sqrt",
    # packed fp32 VALU ops are kept out of every kernel
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
    "-Wall",
]


def bind_command(out: str) -> list[str]:
    """The g++ line of the Python binding for the torch and the Python that run this."""
    import sysconfig

    import torch

    lib = os.path.join(os.path.dirname(torch.__file__), "lib")
    inc = os.path.join(os.path.dirname(torch.__file__), "include")
    return [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-fPIC", "-shared", "-Wall", "-Wno-unused-function",
            "-DUSE_ROCM", "-D__HIP_PLATFORM_AMD__", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
            "-I", os.path.join(ROOT, "include"), "-I", inc, "-I", os.path.join(inc, "torch", "csrc", "api", "include"),
            "-isystem", os.path.join(os.environ.get("ROCM_PATH", "/opt/rocm"), "include"),
            "-I", sysconfig.get_paths()["include"], os.path.join(CSRC, BIND), "-o", out,
            "-L", lib, "-ltorch_python", "-ltorch_cpu", "-lc10", "-lc10_hip"]


def build(verbose: bool = False) -> str:
    """Compile every translation unit in parallel, then link the shared library; the Python binding beside them.
    The library needs hipcc alone: it is in place before a failure of the binding is raised, and without torch the
    binding, which only torch loads, is left out."""
    objdir = os.path.join(HERE, "_build")
    os.makedirs(objdir, exist_ok=True)
    inc = ["-I", os.path.join(ROOT, "include"), "-I", CSRC]
    procs = []
    objs = []
    for src in SOURCES:
        obj = os.path.join(objdir, os.path.splitext(src)[0] + ".o")
        objs.append(obj)
        cmd = [HIPCC, *FLAGS, *inc, "-c", os.path.join(CSRC, src), "-o", obj]
        if verbose:
            print(" ".join(cmd), flush=True)
        procs.append((src, subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT,
                                            text=True)))
    bind, missing = None, None
    try:
        cmd = bind_command(BIND_LIB + ".tmp")
        if verbose:
            print(" ".join(cmd), flush=True)
        bind = subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)
    except (ImportError, OSError) as e:      # no torch, one that does not load, or no C++ compiler
        if getattr(e, "name", None) == "torch":
            print(f"no torch: {os.path.basename(BIND_LIB)} is not built", file=sys.stderr, flush=True)
        else:
            missing = e
    failed = []
    for src, p in procs:
        out, _ = p.communicate()
        if p.returncode != 0:
            failed.append(src)
            sys.stderr.write(out)
    bound = bind.communicate()[0] if bind else ""
    if failed:
        raise RuntimeError(f"hipcc failed for {failed}")
    cmd = [HIPCC, f"--offload-arch={ARCH}", "-shared", "-fPIC", *objs, "-o", LIB + ".tmp"]
    if verbose:
        print(" ".join(cmd), flush=True)
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        sys.stderr.write(res.stdout + res.stderr)
        raise RuntimeError(f"link failed ({res.returncode})")
    os.replace(LIB + ".tmp", LIB)
    if missing or (bind and bind.returncode != 0):
        sys.stderr.write(bound)
        raise RuntimeError(f"the library is built, its binding {BIND} is not") from missing
    if bind:
        os.replace(BIND_LIB + ".tmp", BIND_LIB)
    return LIB


if __name__ == "__main__":
    print(build(verbose=True))
