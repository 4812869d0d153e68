"""Builds libw4b200.so (the sm_100a CUDA library) in-tree with nvcc.

The shared object lands next to this file so that it ships with the source
tree; object files go to ``_build/`` beside it. Only sm_100a is targeted.
_w4torch.so, the small extension module that passes torch tensors to that
library, is built beside it with the host compiler against torch's headers.
"""
from __future__ import annotations

import os
import shutil
import subprocess
import sysconfig
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

PKG_DIR = Path(__file__).resolve().parent
REPO_DIR = PKG_DIR.parent
CSRC = PKG_DIR / "csrc"
BUILD_DIR = PKG_DIR / "_build"
LIB_PATH = PKG_DIR / "libw4b200.so"
TORCH_MODULE_PATH = PKG_DIR / "_w4torch.so"
SOURCES = ["w4_api.cu", "w4_pack.cu", "w4_gemv.cu", "w4_gemv_ops.cu", "w4_gemv_fused.cu",
           "w4_decode.cu", "w4_mega.cu",
           "w4_gemm.cu", "w4_gptq.cu", "w4_tune.cu",
           "w4_kv8.cu", "w4_kv8_attn.cu", "w4_kv8_prompt.cu"]
ARCH_FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a"]


def nvcc_path() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and Path(cand).exists():
            return cand
    raise RuntimeError("nvcc not found: set NVCC or put the CUDA toolkit on PATH")


def common_flags() -> list[str]:
    return ARCH_FLAGS + [
        "-O3", "-lineinfo", "-std=c++17", "--expt-relaxed-constexpr",
        "-Xcompiler", "-fPIC,-O3", f"-I{REPO_DIR / 'include'}", f"-I{CSRC}",
    ]


def _stale(target: Path, deps: list[Path]) -> bool:
    if not target.exists():
        return True
    t = target.stat().st_mtime
    return any(d.stat().st_mtime > t for d in deps)


def build_library(verbose: bool = False, force: bool = False, ptxas_verbose: bool = False) -> Path:
    """Compiles every CUDA source and links libw4b200.so; returns its path."""
    BUILD_DIR.mkdir(exist_ok=True)
    nvcc = nvcc_path()
    headers = sorted(CSRC.glob("*.cuh")) + sorted(CSRC.glob("*.h")) + [REPO_DIR / "include" / "w4b200.h"]
    objs = []
    jobs = []
    for src in SOURCES:
        s = CSRC / src
        o = BUILD_DIR / (src + ".o")
        objs.append(o)
        if force or _stale(o, [s] + headers):
            cmd = [nvcc, *common_flags(), "-c", str(s), "-o", str(o)]
            if ptxas_verbose:
                cmd += ["-Xptxas", "-v"]
            jobs.append(cmd)

    def run(cmd):
        if verbose:
            print(" ".join(cmd), flush=True)
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"nvcc failed ({' '.join(cmd)}):\n{r.stdout}\n{r.stderr}")
        return r.stdout + r.stderr

    with ThreadPoolExecutor(max_workers=min(8, max(1, len(jobs)))) as ex:
        for out in ex.map(run, jobs):
            if (verbose or ptxas_verbose) and out.strip():
                print(out)
    if force or jobs or _stale(LIB_PATH, objs):
        run([nvcc, *ARCH_FLAGS, "-shared", "-Xcompiler", "-fPIC", *map(str, objs),
             "-o", str(LIB_PATH)])
    return LIB_PATH


def build_torch_module(verbose: bool = False, force: bool = False) -> Path:
    """Compiles and links _w4torch.so; returns its path. Needs libw4b200.so.

    It is rebuilt when its sources are newer, and when it was built for another
    torch or Python than this one (BUILD_DIR keeps what it was built for).
    """
    import torch
    from torch.utils import cpp_extension

    src = CSRC / "w4_torch.cpp"
    built_for = BUILD_DIR / "w4torch.built_for"
    version = f"{torch.__version__} {sysconfig.get_config_var('SOABI')}"
    if (not force and built_for.exists() and built_for.read_text() == version and
            not _stale(TORCH_MODULE_PATH, [src, REPO_DIR / "include" / "w4b200.h"])):
        return TORCH_MODULE_PATH
    BUILD_DIR.mkdir(exist_ok=True)
    cuda = Path(nvcc_path()).resolve().parent.parent
    torch_lib = Path(torch.__file__).resolve().parent / "lib"
    cmd = ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-w",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
           f'-DW4_TORCH_VERSION="{torch.__version__}"',
           *(f"-isystem{p}" for p in cpp_extension.include_paths()),
           f"-isystem{sysconfig.get_paths()['include']}", f"-isystem{cuda / 'include'}", str(src),
           "-o", str(TORCH_MODULE_PATH), f"-L{PKG_DIR}", "-l:libw4b200.so", f"-L{torch_lib}",
           "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch_cuda", "-ltorch", "-ltorch_python",
           "-Wl,-rpath,$ORIGIN"]
    if verbose:
        print(" ".join(cmd), flush=True)
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"{cmd[0]} failed ({' '.join(cmd)}):\n{r.stdout}\n{r.stderr}")
    built_for.write_text(version)
    return TORCH_MODULE_PATH


if __name__ == "__main__":
    import sys

    print(build_library(verbose=True, force="--force" in sys.argv,
                        ptxas_verbose="-v" in sys.argv))
    print(build_torch_module(verbose=True, force="--force" in sys.argv))
