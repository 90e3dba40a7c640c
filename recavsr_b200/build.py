"""Build librecavsr_b200.so (the C-ABI library) in-tree with nvcc for sm_100a.

    python -m recavsr_b200.build          # incremental
    python -m recavsr_b200.build --force  # rebuild everything

Objects go to recavsr_b200/_build/, the library to recavsr_b200/librecavsr_b200.so
and the Python binding of the block-scaled FP8 operators (a CPython extension on
torch's C++ headers, linked to the library) to recavsr_b200/_fp8_block.so.
The CUDA runtime is linked statically; the driver is reached through
cudaGetDriverEntryPoint, so the library needs no -lcuda at link time.
"""
from __future__ import annotations

import argparse
import concurrent.futures as cf
import importlib.metadata
import os
import shutil
import subprocess
import sysconfig

PKG = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(PKG, "csrc")
OBJ = os.path.join(PKG, "_build")
LIB = os.path.join(PKG, "librecavsr_b200.so")
BINDING = os.path.join(PKG, "_fp8_block.so")
BINDING_KEY = os.path.join(OBJ, "_fp8_block.key")
BINDING_SOURCE = os.path.join(CSRC, "fp8_block_torch.cpp")
INCLUDE = os.path.join(os.path.dirname(PKG), "include", "recavsr_b200.h")
SOURCES = ["runtime.cu", "quant.cu", "glue.cu", "gemm.cu", "attention.cu", "session.cu", "pipeline.cu", "decoder_attention.cu", "decoder.cu", "colorfix.cu",
           "fp8_block.cu", "fp8_block_gemm.cu"]
HEADERS = ["common.cuh", "sm100.cuh", "fp8_block.cuh"]
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
FLAGS = ["-O3", "-std=c++17", "-lineinfo", "-Xcompiler", "-fPIC", "-Xcompiler", "-O2",
         "--expt-relaxed-constexpr", "-diag-suppress", "177"]


def nvcc() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found: the recavsr_b200 library must be built with CUDA 12.9+")


def _stale(target: str, deps: list[str]) -> bool:
    if not os.path.exists(target):
        return True
    t = os.path.getmtime(target)
    return any(os.path.getmtime(d) > t for d in deps)


def _compile(src: str, force: bool) -> str:
    obj = os.path.join(OBJ, src.replace(".cu", ".o"))
    deps = [os.path.join(CSRC, src)] + [os.path.join(CSRC, h) for h in HEADERS]
    if force or _stale(obj, deps):
        cmd = [nvcc(), *ARCH, *FLAGS, "-c", os.path.join(CSRC, src), "-o", obj]
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode:
            raise RuntimeError(f"nvcc failed for {src}:\n{r.stderr}")
    return obj


def _binding_key() -> str:
    """What the binding's object layouts depend on besides its own sources."""
    return f"torch {importlib.metadata.version('torch')}, {sysconfig.get_config_var('SOABI')}"


def _build_binding(force: bool) -> None:
    try:
        with open(BINDING_KEY) as f:
            built_for = f.read()
    except OSError:
        built_for = None
    key = _binding_key()
    if not force and built_for == key and not _stale(BINDING, [BINDING_SOURCE, INCLUDE]):
        return
    import torch

    root = os.path.dirname(torch.__file__)
    cuda = os.path.join(os.path.dirname(os.path.dirname(os.path.realpath(nvcc()))), "include")
    include = [os.path.join(root, "include"), os.path.join(root, "include", "torch", "csrc", "api", "include"),
               sysconfig.get_paths()["include"], cuda]
    part = BINDING + ".part"          # whole before it has its name: another process may be importing
    # The host compiler that nvcc uses, not $CXX: one with a C++ runtime of its
    # own linked in clashes with the runtime torch has loaded.
    cmd = ["g++", "-O2", "-std=c++17", "-shared", "-fPIC",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", *(f"-I{d}" for d in include),
           BINDING_SOURCE, "-o", part, "-L" + os.path.join(root, "lib"), "-ltorch_python", "-ltorch_cpu",
           "-ltorch_cuda", "-lc10", "-lc10_cuda", "-L" + PKG, "-l:" + os.path.basename(LIB), "-Wl,-rpath,$ORIGIN"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode:
        raise RuntimeError(f"{cmd[0]} failed for {os.path.basename(BINDING_SOURCE)}:\n{r.stderr}")
    os.replace(part, BINDING)
    with open(BINDING_KEY, "w") as f:
        f.write(key)


def build(force: bool = False, verbose: bool = False) -> str:
    os.makedirs(OBJ, exist_ok=True)
    with cf.ThreadPoolExecutor(max_workers=min(8, os.cpu_count() or 1)) as ex:
        objs = list(ex.map(lambda s: _compile(s, force), SOURCES))
    if force or _stale(LIB, objs):
        cmd = [nvcc(), *ARCH, "-shared", "-cudart", "static", "-o", LIB, *objs]
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode:
            raise RuntimeError(f"link failed:\n{r.stderr}")
    _build_binding(force)
    if verbose:
        print(LIB)
    return LIB


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--force", action="store_true")
    build(ap.parse_args().force, verbose=True)
