"""Builds ``libtopos_b200.so`` in-tree with nvcc for sm_100a, and ``_operators.so``, the binding of
its device operators to torch tensors.

Host files (``csrc/*.cpp``) and CUDA files (``csrc/*.cu``) compile to objects
under ``_build/`` in parallel, then link into one shared library with a static
CUDA runtime, the driver API and NVRTC.  NCCL is loaded at run time.
"""
from __future__ import annotations

import concurrent.futures as cf
import glob
import importlib.metadata
import importlib.util
import os
import subprocess
import sys
import sysconfig
from typing import Optional

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
CSRC = os.path.join(HERE, "csrc")
BUILD = os.path.join(ROOT, "_build")
OUT = os.path.join(HERE, "libtopos_b200.so")
BINDING = os.path.join(HERE, "_operators.so")
BINDING_STAMP = os.path.join(HERE, "_operators.stamp")
NVCC = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
COMMON = ["-O3", "-std=c++17", "-lineinfo", "-Xcompiler", "-fPIC,-ffp-contract=off",
          f"-I{os.path.join(ROOT, 'include')}", "-I/usr/local/cuda/include"]


def _compile(src: str) -> str:
    obj = os.path.join(BUILD, os.path.basename(src) + ".o")
    deps = [src] + glob.glob(os.path.join(CSRC, "*.h")) + [os.path.join(ROOT, "include", "topos_b200.h")]
    if os.path.exists(obj) and os.path.getmtime(obj) >= max(os.path.getmtime(d) for d in deps):
        return obj
    cmd = [NVCC, *ARCH, *COMMON, "-c", src, "-o", obj]
    if src.endswith(".cu"):
        cmd += ["-Xptxas", "-v"] if os.environ.get("TB_PTXAS_VERBOSE") else []
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"nvcc failed on {src}:\n{res.stdout}\n{res.stderr}")
    if res.stderr.strip() and os.environ.get("TB_PTXAS_VERBOSE"):
        sys.stderr.write(res.stderr)
    return obj


def build_binding(force: bool = False) -> Optional[str]:
    """Compiles ``csrc/python/operators_binding.cpp`` against torch and the library; where there is no
    torch, nothing, for then nobody has a tensor to pass."""
    spec = importlib.util.find_spec("torch")
    if spec is None or spec.origin is None:
        return None
    torch = os.path.dirname(spec.origin)
    # another torch or Python has another layout, whatever the files' times say
    stamp = f"torch {importlib.metadata.version('torch')} in {torch}, Python {sys.version}\n"
    src = os.path.join(CSRC, "python", "operators_binding.cpp")
    deps = [src, os.path.join(ROOT, "include", "topos_b200.h")]
    if (not force and os.path.exists(BINDING) and _text(BINDING_STAMP) == stamp
            and os.path.getmtime(BINDING) >= max(os.path.getmtime(d) for d in deps)):
        return BINDING
    cmd = ["g++", "-O2", "-std=c++17", "-shared", "-fPIC", "-w", src, "-o", BINDING,
           f"-I{os.path.join(torch, 'include')}", f"-I{sysconfig.get_paths()['include']}",
           "-I/usr/local/cuda/include", f"-L{os.path.join(torch, 'lib')}", "-ltorch_python", "-ltorch",
           "-ltorch_cpu", "-ltorch_cuda", "-lc10", "-lc10_cuda",
           f"-L{HERE}", "-l:libtopos_b200.so", "-Wl,-rpath,$ORIGIN",
           f"-Wl,-rpath,{os.path.join(torch, 'lib')}"]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"g++ failed on {src}:\n{res.stdout}\n{res.stderr}")
    with open(BINDING_STAMP, "w") as f:
        f.write(stamp)
    return BINDING


def _text(path: str) -> str:
    try:
        with open(path) as f:
            return f.read()
    except OSError:
        return ""


def build(force: bool = False) -> str:
    out = build_library(force)
    build_binding(force)
    return out


def build_library(force: bool = False) -> str:
    os.makedirs(BUILD, exist_ok=True)
    sources = sorted(glob.glob(os.path.join(CSRC, "*.cpp")) + glob.glob(os.path.join(CSRC, "*.cu")))
    if force:
        for obj in glob.glob(os.path.join(BUILD, "*.o")):
            os.remove(obj)
    with cf.ThreadPoolExecutor(max_workers=min(8, len(sources))) as pool:
        objects = list(pool.map(_compile, sources))
    if (not force and os.path.exists(OUT)
            and os.path.getmtime(OUT) >= max(os.path.getmtime(o) for o in objects)):
        return OUT
    cmd = [NVCC, *ARCH, "-shared", "-o", OUT, *objects, "-L/usr/local/cuda/lib64",
           "-lnvrtc", "-ldl", "-cudart", "static"]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"link failed:\n{res.stdout}\n{res.stderr}")
    return OUT


if __name__ == "__main__":
    print(build(force="--force" in sys.argv))
