"""Build recipe of libh24.so (the CUDA library behind pollux_b200) and of
the module _h24_torch (the short way from torch tensors to its decoding-step
calls).

    python -m pollux_b200.build          # compiles into pollux_b200/_lib/

Every CUDA source is compiled for sm_100a only
(``-gencode arch=compute_100a,code=sm_100a``) with line info, and linked with
the static CUDA runtime so that the library does not depend on which
libcudart the host process (e.g. torch) has loaded.
"""
from __future__ import annotations

import concurrent.futures as cf
import os
import shutil
import subprocess
import sys
import sysconfig
import warnings

from ._native import torch_module_path

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
OUT_DIR = os.path.join(HERE, "_lib")
BUILD_DIR = os.path.join(HERE, "_build")
LIB = os.path.join(OUT_DIR, "libh24.so")
TORCH_SRC = os.path.join(CSRC, "h24_torch.cpp")
HEADER = os.path.join(os.path.dirname(HERE), "include", "h24.h")
SOURCES = ["h24_capi.cu", "h24_pack.cu", "h24_dequant.cu", "h24_lut.cu", "h24_int8.cu", "h24_int8_rows.cu", "h24_int8_linear.cu", "h24_sample.cu", "h24_norm.cu", "h24_ce.cu", "h24_project.cu", "h24_rowrms.cu", "h24_search.cu", "h24_codebook.cpp"]
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
NVCC_FLAGS = ARCH + ["-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC,-O3",
                     "--expt-relaxed-constexpr", "-Werror", "all-warnings"]


def nvcc() -> str:
    for cand in (os.environ.get("NVCC"), "/usr/local/cuda/bin/nvcc", shutil.which("nvcc")):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found")


def _stale(target: str, deps: list[str]) -> bool:
    if not os.path.exists(target):
        return True
    t = os.path.getmtime(target)
    return any(os.path.getmtime(d) > t for d in deps)


def _run(cmd: list[str]) -> str:
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"compilation failed: {' '.join(cmd)}\n{r.stdout}\n{r.stderr}")
    return r.stdout + r.stderr


def torch_command(src: str, out: str) -> list[str]:
    """g++ command of _h24_torch.  torch's libraries are in the process that
    loads the module; nothing but their names is recorded."""
    import torch
    root = os.path.dirname(torch.__file__)
    cuda = os.path.join(os.path.dirname(os.path.dirname(nvcc())), "include")
    inc = [os.path.join(root, "include"), os.path.join(root, "include", "torch", "csrc", "api", "include"), cuda]
    return ["g++", "-O2", "-std=c++17", "-shared", "-fPIC", "-Wall", "-Werror", src, "-o", out,
            "-I" + sysconfig.get_paths()["include"]] + [x for d in inc for x in ("-isystem", d)] + \
           ["-L" + os.path.join(root, "lib"), "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch_cuda", "-ltorch_python"]


def build_torch_module() -> str:
    """Compile (if stale) _h24_torch for this torch and interpreter and return its path."""
    path = torch_module_path()
    if _stale(path, [TORCH_SRC, HEADER]):
        os.makedirs(OUT_DIR, exist_ok=True)
        part = f"{path}.{os.getpid()}"
        try:
            _run(torch_command(TORCH_SRC, part))
            os.replace(part, path)
        finally:
            if os.path.exists(part):
                os.remove(part)
    return path


def build(verbose: bool = False, ptxas_info: bool = False) -> str:
    """Compile (incrementally) and return the path of libh24.so.  _h24_torch is
    built beside it; a failure of that is a warning, since libh24 runs without it."""
    os.makedirs(OUT_DIR, exist_ok=True)
    os.makedirs(BUILD_DIR, exist_ok=True)
    headers = [os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith((".cuh", ".h"))]
    headers.append(HEADER)
    objs, jobs = [], []
    for src in SOURCES:
        path = os.path.join(CSRC, src)
        obj = os.path.join(BUILD_DIR, src + ".o")
        objs.append(obj)
        if _stale(obj, [path] + headers) or ptxas_info:
            cmd = [nvcc()] + NVCC_FLAGS + (["-Xptxas", "-v"] if ptxas_info else []) + \
                  ["-c", path, "-o", obj]
            jobs.append(cmd)
    with cf.ThreadPoolExecutor(max_workers=len(jobs) + 1) as ex:
        torch_module = ex.submit(build_torch_module)
        for out in ex.map(_run, jobs):
            if verbose and out.strip():
                print(out)
        if jobs or _stale(LIB, objs):
            _run([nvcc()] + ARCH + ["-shared", "-cudart", "static", "-o", LIB] + objs)
        try:
            torch_module.result()
        except Exception as e:  # a torch without CUDA's headers or libraries, or none
            warnings.warn(f"_h24_torch was not built: {e}", RuntimeWarning)
    return LIB


if __name__ == "__main__":
    path = build(verbose=True, ptxas_info="-v" in sys.argv)
    print(path)
