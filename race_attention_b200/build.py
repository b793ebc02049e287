"""Builds librace_b200.so in-tree with nvcc for sm_100a, and _race_torch.so, the
torch bindings of its 8-bit operators, with g++.

    python -m race_attention_b200.build      (or __graft_entry__.build())

The translation units compile in parallel; the results land next to
this file so they travel with the source tree.
"""
from __future__ import annotations

import concurrent.futures as cf
import os
import shutil
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
CSRC = os.path.join(HERE, "csrc")
OUT = os.path.join(HERE, "librace_b200.so")
OUT_TORCH = os.path.join(HERE, "_race_torch.so")   # torch bindings of the 8-bit operators
SOURCES = ["race_capi.cu", "race_f32_d32.cu", "race_f32_d64.cu", "race_bf16_d32.cu",
           "race_bf16_d64.cu", "race_probs.cu", "race_comm.cu", "race_norm.cu", "race_quant.cu",
           "race_matmul.cu", "race_adamw.cu"]
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
FLAGS = ["-O3", "-std=c++17", "-lineinfo", "-Xcompiler", "-fPIC", "--expt-relaxed-constexpr",
         "-I" + os.path.join(ROOT, "include"), "-I" + CSRC]


def nvcc() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found")


def _stale() -> bool:
    if not os.path.exists(OUT) or not os.path.exists(OUT_TORCH):
        return True
    t = min(os.path.getmtime(OUT), os.path.getmtime(OUT_TORCH))
    hdr = os.path.join(ROOT, "include", "race_b200.h")
    deps = [os.path.join(CSRC, f) for f in os.listdir(CSRC)] + [hdr, os.path.abspath(__file__)]
    return any(os.path.getmtime(p) > t for p in deps)


def _compile_torch(obj: str, force: bool) -> str:
    """The bindings are plain C++ over the C entry points: no device code."""
    import sysconfig

    from torch.utils.cpp_extension import include_paths
    src = os.path.join(CSRC, "race_torch.cpp")
    newest = max(os.path.getmtime(src), os.path.getmtime(os.path.join(ROOT, "include", "race_b200.h")))
    if force or not os.path.exists(obj) or os.path.getmtime(obj) < newest:
        cuda = os.path.join(os.path.dirname(os.path.dirname(os.path.realpath(nvcc()))), "include")
        inc = [f"-I{p}" for p in (*include_paths(), sysconfig.get_paths()["include"], cuda,
                                  os.path.join(ROOT, "include"))]
        _run(["g++", "-O2", "-std=c++17", "-fPIC", "-DTORCH_EXTENSION_NAME=_race_torch", *inc, "-c", src,
              "-o", obj], "g++ failed on race_torch.cpp")
    return obj


def _link_torch(obj: str) -> None:
    import torch
    libs = os.path.join(os.path.dirname(torch.__file__), "lib")
    tmp = OUT_TORCH + ".tmp"
    _run(["g++", "-shared", "-o", tmp, obj, "-L" + libs, "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch_cuda",
          "-ltorch", "-ltorch_python", "-L" + HERE, "-lrace_b200", "-Wl,-rpath,$ORIGIN"], "link failed")
    os.replace(tmp, OUT_TORCH)


def _run(cmd, what: str) -> None:
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"{what}:\n{r.stderr}")


def build(force: bool = False, verbose: bool = False) -> str:
    if not force and not _stale():
        return OUT
    objdir = os.path.join(HERE, "_build")
    os.makedirs(objdir, exist_ok=True)
    cc = nvcc()

    def compile_one(src):
        obj = os.path.join(objdir, src.replace(".cu", ".o"))
        cmd = [cc, *ARCH, *FLAGS, "-c", os.path.join(CSRC, src), "-o", obj]
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"nvcc failed on {src}:\n{r.stderr}")
        if verbose and r.stderr:
            print(r.stderr, file=sys.stderr)
        return obj

    hdrs = [os.path.join(CSRC, f) for f in os.listdir(CSRC) if not f.endswith(".cu")]
    hdrs.append(os.path.join(ROOT, "include", "race_b200.h"))
    newest_hdr = max(os.path.getmtime(h) for h in hdrs)

    def fresh(src):
        obj = os.path.join(objdir, src.replace(".cu", ".o"))
        return (not force and os.path.exists(obj) and
                os.path.getmtime(obj) > max(newest_hdr, os.path.getmtime(os.path.join(CSRC, src))))

    todo = [s for s in SOURCES if not fresh(s)]
    with cf.ThreadPoolExecutor(len(todo) + 1) as ex:
        binding = ex.submit(_compile_torch, os.path.join(objdir, "race_torch.o"), force)
        list(ex.map(compile_one, todo))
        torch_obj = binding.result()
    objs = [os.path.join(objdir, s.replace(".cu", ".o")) for s in SOURCES]
    tmp = OUT + ".tmp"
    cmd = [cc, *ARCH, "-shared", "-o", tmp, *objs, "-ldl"]   # cudart linked statically
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"link failed:\n{r.stderr}")
    os.replace(tmp, OUT)
    _link_torch(torch_obj)
    return OUT


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="-v" in sys.argv))
