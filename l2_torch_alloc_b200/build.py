"""Builds sideaware.so (the C-ABI library) in place with nvcc for sm_100a.

    python -m l2_torch_alloc_b200.build [--force]
    python -m l2_torch_alloc_b200.build --alloc-only    # sideaware_alloc.so: allocator and topology only
                                                          (include/sideaware_alloc.h; the counterpart of the
                                                          reference's sideaware_alloc.cu for non-PyTorch projects)

No GPU is needed to build.  The library links the CUDA runtime statically and
loads libcuda.so.1 / libnvrtc at run time, so it can be opened (not used) on a
machine without a driver.
"""
from __future__ import annotations

import os
import shutil
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
GEN = os.path.join(CSRC, "_gen")
OUT = os.path.join(HERE, "sideaware.so")
OUT_ALLOC = os.path.join(HERE, "sideaware_alloc.so")

SOURCES = ["sa_api.cpp", "sa_context.cpp", "sa_alloc.cpp", "sa_driver.cpp", "sa_jit.cpp", "sa_topology.cpp",
           "sa_probe.cu", "sa_kernels.cu", "sa_memcpy_bulk.cu", "sa_rope_bulk.cu",
           "sa_ops_api.cpp", "sa_rope_axes.cu", "sa_group_norm.cu", "sa_dropout.cu"]
ALLOC_ONLY_SOURCES = ["sa_api.cpp", "sa_context.cpp", "sa_alloc.cpp", "sa_driver.cpp", "sa_topology.cpp", "sa_probe.cu"]
EMBEDDED = [("kSaSchedSource", "sa_sched.cuh"), ("kSaJitTemplateSource", "sa_jit_template.cuh")]


def nvcc_path() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found (set NVCC)")


def generate_embedded() -> str:
    """Device headers that NVRTC needs at run time, as C++ raw string literals."""
    os.makedirs(GEN, exist_ok=True)
    parts = ["// generated by build.py from the .cuh files beside it - do not edit\n"]
    for name, fn in EMBEDDED:
        text = open(os.path.join(CSRC, fn)).read().replace("#pragma once\n", "")
        assert ')SA_EMBED"' not in text
        parts.append(f'static const char {name}[] = R"SA_EMBED({text})SA_EMBED";\n')
    path = os.path.join(GEN, "sa_embedded_sources.inc")
    new = "".join(parts)
    if not os.path.exists(path) or open(path).read() != new:
        with open(path, "w") as f:
            f.write(new)
    return path


def needs_build(out: str) -> bool:
    if not os.path.exists(out):
        return True
    t = os.path.getmtime(out)
    deps = [os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith((".cu", ".cpp", ".hpp", ".cuh"))]
    deps += [os.path.join(HERE, "..", "include", "sideaware.h"), os.path.abspath(__file__)]
    return any(os.path.getmtime(d) > t for d in deps)


def build(force: bool = False, verbose: bool = False, alloc_only: bool = False) -> str:
    generate_embedded()
    out = OUT_ALLOC if alloc_only else OUT
    if not force and not needs_build(out):
        return out
    cmd = [nvcc_path(), "-gencode", "arch=compute_100a,code=sm_100a", "-lineinfo", "-O3", "-std=c++17",
           "-Xcompiler", "-fPIC,-fvisibility=hidden,-Wall,-ffp-contract=off", "-shared", "-cudart", "static"]
    if alloc_only:
        cmd += ["-DSIDEAWARE_ALLOC_ONLY"]
    if verbose:
        cmd += ["-Xptxas", "-v"]
    cmd += [os.path.join(CSRC, s) for s in (ALLOC_ONLY_SOURCES if alloc_only else SOURCES)]
    cmd += ["-o", out, "-ldl", "-lpthread"]
    subprocess.check_call(cmd, cwd=CSRC)
    return out


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="-v" in sys.argv, alloc_only="--alloc-only" in sys.argv))
