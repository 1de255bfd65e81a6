"""Builds mlx3d_amd/libgsx.so from the HIP sources for gfx950.

Each translation unit is compiled with hipcc in parallel, then linked into
one shared library in the package directory (in-tree, so it travels with
the source tree).  Flags:
  -ffp-contract=off          every float op rounded on its own (bit-exact
                             radii, tile rectangles, contributor counts)
  -munsafe-fp-atomics        hardware global_atomic_add_f32 in the backward
  -packed-fp32-ops disabled  no v_pk_*_f32 generated
Beside it goes mlx3d_amd/_autograd.so, the field layers' autograd nodes: host code
against torch's headers, linked to libgsx.so.
The compiler's per-kernel resource usage (VGPRs, scratch, occupancy) is
written to _build/resource_usage.json, and the build fails if any kernel
spills registers to scratch memory.
"""

from __future__ import annotations

import concurrent.futures
import json
import os
import re
import subprocess
import sys
import sysconfig

HERE = os.path.dirname(os.path.abspath(__file__))
PKG = os.path.dirname(HERE)
ROOT = os.path.dirname(PKG)
SOURCES = ["capi.hip", "preprocess.hip", "binning.hip", "raster.hip", "train.hip", "mesh.hip",
           "density.hip", "geometry.hip", "feedforward.hip", "distil.hip",
           "embedding.hip", "layernorm.hip", "dropout.hip"]
LIB = os.path.join(PKG, "libgsx.so")
AUTOGRAD = os.path.join(PKG, "_autograd.so")
ARCH = os.environ.get("GSX_OFFLOAD_ARCH", "gfx950")

HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
FLAGS = [
    "-O3", "-std=c++17", "-fPIC", f"--offload-arch={ARCH}",
    "-ffp-contract=off", "-munsafe-fp-atomics",
    "-fno-gpu-flush-denormals-to-zero",
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
    "-Wall", "-Wno-unused-function",
    f"-I{os.path.join(ROOT, 'include')}", f"-I{HERE}",
]


_REMARK = "-Rpass-analysis=kernel-resource-usage"


def _resources(stderr: str) -> dict:
    """{kernel: {VGPRs, AGPRs, ScratchSize, Occupancy, LDS}} from the
    compiler's kernel-resource-usage remarks."""
    out: dict = {}
    cur = None
    for ln in stderr.splitlines():
        if _REMARK not in ln or "remark:" not in ln:
            continue
        body = ln.split("remark:", 1)[1].replace(f"[{_REMARK}]", "").strip()
        key, _, val = body.partition(":")
        if key == "Function Name":
            cur = out.setdefault(val.strip(), {})
        elif cur is not None:
            name = key.split("[")[0].strip()
            try:
                cur[name] = int(val.strip())
            except ValueError:
                pass
    return out


def _compile(src: str, obj: str) -> dict:
    cmd = [HIPCC, *FLAGS, _REMARK, "-c", os.path.join(HERE, src), "-o", obj]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"hipcc failed for {src}:\n{r.stdout}\n{r.stderr}")
    # The host pass warns that it does not know the packed-fp32 feature;
    # resource-usage remarks are collected, not echoed.
    noise = [ln for ln in r.stderr.splitlines()
             if "packed-fp32-ops" not in ln and _REMARK not in ln and ln.strip()
             and not re.match(r"^\s*\d*\s*\|", ln)]  # the remarks' source excerpts
    if noise:
        sys.stderr.write("\n".join(noise) + "\n")
    return _resources(r.stderr)


def _compile_autograd(obj: str) -> None:
    from torch.utils import cpp_extension

    includes = [*cpp_extension.include_paths(), sysconfig.get_paths()["include"],
                "/opt/rocm/include", os.path.join(ROOT, "include")]
    # (the last two name the runtime that torch's own headers are to declare)
    cmd = ["g++", "-O2", "-std=c++17", "-fPIC", "-Wall", "-Wno-unknown-pragmas",
           *(f"-I{d}" for d in includes), "-D__HIP_PLATFORM_AMD__=1", "-DUSE_ROCM=1",
           "-c", os.path.join(HERE, "autograd.cpp"), "-o", obj]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"g++ failed for autograd.cpp:\n{r.stdout}\n{r.stderr}")


def _link_autograd(obj: str) -> None:
    from torch.utils import cpp_extension

    libs = [f"-L{d}" for d in cpp_extension.library_paths()]
    cmd = ["g++", "-shared", "-o", AUTOGRAD + ".tmp", obj, *libs, "-lc10", "-lc10_hip",
           "-ltorch_cpu", "-ltorch_python", f"-L{PKG}", "-l:libgsx.so", "-Wl,-rpath,$ORIGIN"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"link failed for {AUTOGRAD}:\n{r.stdout}\n{r.stderr}")
    os.replace(AUTOGRAD + ".tmp", AUTOGRAD)


def build(verbose: bool = False) -> str:
    objdir = os.path.join(PKG, "_build")
    os.makedirs(objdir, exist_ok=True)
    objs = [os.path.join(objdir, s.replace(".hip", ".o")) for s in SOURCES]
    nodes = os.path.join(objdir, "autograd.o")
    with concurrent.futures.ThreadPoolExecutor(max_workers=min(8, len(SOURCES))) as ex:
        host = ex.submit(_compile_autograd, nodes)
        usage = list(ex.map(lambda a: _compile(*a), zip(SOURCES, objs)))
        host.result()
    kernels = {k: v for u in usage for k, v in u.items()}
    with open(os.path.join(objdir, "resource_usage.json"), "w") as f:
        json.dump(kernels, f, indent=1, sort_keys=True)
    spills = sorted(k for k, v in kernels.items() if v.get("ScratchSize", 0) > 0)
    if spills:
        raise RuntimeError("kernels spill registers to scratch (ScratchSize > 0): "
                           + ", ".join(spills))
    tmp = LIB + ".tmp"
    cmd = [HIPCC, f"--offload-arch={ARCH}", "-shared", "-fPIC", "-o", tmp, *objs]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"link failed:\n{r.stdout}\n{r.stderr}")
    os.replace(tmp, LIB)
    _link_autograd(nodes)
    if verbose:
        print(f"built {LIB}")
    return LIB


if __name__ == "__main__":
    build(verbose=True)
