"""Build liblewm_b200.so in-tree with nvcc for sm_100a, and the torch extension module
_torch_ops.so (the training operators' torch side) with the host compiler.

    python -m lewm_flash_b200.build
"""

from __future__ import annotations

import os
import shutil
import subprocess
import sys
from pathlib import Path

PKG = Path(__file__).resolve().parent
REPO = PKG.parent
CSRC = PKG / "csrc"
LIB = PKG / "liblewm_b200.so"
SOURCES = ["api.cu", "rollout_kernels.cu", "tile_call.cu", "fp32_path.cu", "icem_kernels.cu", "noalloc.cu", "encoder.cu",
           "train_norm.cu", "train_norm_f32.cu", "train_norm_bf16.cu", "train_norm_f16.cu", "grad_clip.cu"]
HEADERS = ["lewm_common.cuh", "lewm_internal.h", "train_elem.cuh", "train_norm.h", "train_norm.cuh"]
EXT = PKG / "_torch_ops.so"
EXT_SOURCES = ["torch_ops.cpp"]
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]


def nvcc() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and Path(cand).exists():
            return cand
    raise RuntimeError("nvcc not found")


def _stale(target: Path, deps) -> bool:
    if not target.exists():
        return True
    t = target.stat().st_mtime
    return any(d.stat().st_mtime > t for d in deps)


def _run(cmd, target: Path, verbose: bool) -> None:
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"{Path(cmd[0]).name} failed ({res.returncode}):\n{res.stderr[-8000:]}")
    if verbose:
        sys.stderr.write(res.stderr)
    os.replace(str(target) + ".tmp", target)


def build(force: bool = False, verbose: bool = False) -> Path:
    header = REPO / "include" / "lewm_b200.h"
    if force or _stale(LIB, [CSRC / s for s in SOURCES + HEADERS] + [header, Path(__file__)]):
        cmd = [nvcc(), *ARCH, "-O3", "-std=c++17", "--threads", "0", "-lineinfo", "-shared", "-Xcompiler", "-fPIC",
               "-Xcompiler", "-fvisibility=hidden", "--expt-relaxed-constexpr",
               "-I", str(REPO / "include"), "-o", str(LIB) + ".tmp"]
        if verbose:
            cmd += ["-Xptxas", "-v"]
        _run(cmd + [str(CSRC / s) for s in SOURCES], LIB, verbose)
    if force or _stale(EXT, [CSRC / s for s in EXT_SOURCES] + [header, Path(__file__)]):
        _build_ext(verbose)
    return LIB


def _build_ext(verbose: bool) -> None:
    import sysconfig

    import torch

    tdir = Path(torch.__file__).parent
    cuda = Path(nvcc()).resolve().parents[1]
    inc = [tdir / "include", tdir / "include" / "torch" / "csrc" / "api" / "include",
           sysconfig.get_paths()["include"], cuda / "include"]
    cmd = [shutil.which("g++") or "g++", "-O2", "-std=c++17", "-shared", "-fPIC", "-fvisibility=hidden",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch.compiled_with_cxx11_abi())}", "-I", str(REPO / "include")]
    for d in inc:
        cmd += ["-isystem", str(d)]
    cmd += ["-o", str(EXT) + ".tmp", *[str(CSRC / s) for s in EXT_SOURCES], "-L", str(PKG), "-llewm_b200",
            "-L", str(tdir / "lib"), "-ltorch", "-ltorch_cpu", "-ltorch_cuda", "-ltorch_python", "-lc10", "-lc10_cuda",
            "-Wl,-rpath,$ORIGIN"]
    _run(cmd, EXT, verbose)


if __name__ == "__main__":
    build(force="--force" in sys.argv, verbose="-v" in sys.argv)
    print(LIB)
