"""Build ``libtorque_b200.so`` (the C-ABI CUDA library) in-tree with nvcc, and
``_torch_bind.so`` (the native Python binding of its serving operators on torch
tensors) with g++.

    python -m torque_mlx_b200.build            # or build_library() from Python

The library is compiled for sm_100a only and placed next to this file so it
travels with the source tree; it is loaded by ``torque_mlx_b200._lib``.
"""

from __future__ import annotations

import os
import shutil
import subprocess
import sys
from pathlib import Path

PKG = Path(__file__).resolve().parent
CSRC = PKG / "csrc"
LIB = PKG / "libtorque_b200.so"
BIND = PKG / "_torch_bind.so"
SOURCES = ["tq_append.cu", "tq_decode.cu", "tq_decode_mma.cu", "tq_glue.cu", "tq_paged.cu",
           "tq_paged_attend.cu", "tq_paged_prefill.cu", "tq_peer.cu", "tq_verify.cu", "tq_w4.cu"]
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]


def _nvcc() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and Path(cand).exists():
            return cand
    raise RuntimeError("nvcc not found: the CUDA toolkit is required to build libtorque_b200.so")


def _stale() -> bool:
    if not LIB.exists() or not BIND.exists():
        return True
    t = min(LIB.stat().st_mtime, BIND.stat().st_mtime)
    deps = [*CSRC.glob("*.cu"), *CSRC.glob("*.cuh"), *CSRC.glob("*.cpp"), *(PKG.parent / "include").glob("*.h")]
    return any(p.stat().st_mtime > t for p in deps)


def _binding_commands(objdir: Path) -> tuple[list[str], list[str]]:
    """The compile and the link command of ``_torch_bind.so``."""
    import sysconfig

    import torch

    torch_dir = Path(torch.__file__).resolve().parent
    cuda = Path(_nvcc()).resolve().parent.parent
    obj = objdir / "tq_torch.o"
    includes = [torch_dir / "include", torch_dir / "include" / "torch" / "csrc" / "api" / "include",
                Path(sysconfig.get_paths()["include"]), cuda / "include"]
    compile_cmd = [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-fPIC",
                   f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
                   *[f"-I{p}" for p in includes], "-c", str(CSRC / "tq_torch.cpp"), "-o", str(obj)]
    link_cmd = [compile_cmd[0], "-shared", str(obj), "-o", str(BIND) + ".tmp", f"-L{PKG}", f"-l:{LIB.name}",
                f"-L{torch_dir / 'lib'}", "-ltorch_python", "-ltorch", "-ltorch_cpu", "-ltorch_cuda", "-lc10",
                "-lc10_cuda", f"-L{cuda / 'lib64'}", "-lcudart", "-Wl,-rpath,$ORIGIN"]
    return compile_cmd, link_cmd


def build_library(force: bool = False, verbose: bool = False) -> Path:
    """Compile every source to an object in parallel, then link the shared library."""
    if not force and not _stale():
        return LIB
    from concurrent.futures import ThreadPoolExecutor

    nvcc = _nvcc()
    objdir = PKG / "_build"
    objdir.mkdir(exist_ok=True)
    common = [*ARCH, "-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC", "--expt-relaxed-constexpr",
              "-I", str(PKG.parent / "include")]
    if verbose:
        common.append("-Xptxas=-v")

    def compile_one(src: str) -> Path:
        obj = objdir / (Path(src).stem + ".o")
        cmd = [nvcc, *common, "-c", str(CSRC / src), "-o", str(obj)]
        res = subprocess.run(cmd, capture_output=True, text=True)
        if verbose or res.returncode:
            sys.stderr.write(res.stdout + res.stderr)
        if res.returncode:
            raise RuntimeError(f"nvcc failed on {src}")
        return obj

    def run(cmd: list[str], what: str) -> None:
        res = subprocess.run(cmd, capture_output=True, text=True)
        if verbose or res.returncode:
            sys.stderr.write(res.stdout + res.stderr)
        if res.returncode:
            raise RuntimeError(f"{cmd[0]} failed on {what}")

    bind_compile, bind_link = _binding_commands(objdir)
    with ThreadPoolExecutor(max_workers=len(SOURCES) + 1) as pool:
        binding = pool.submit(run, bind_compile, "tq_torch.cpp")
        objs = list(pool.map(compile_one, SOURCES))
        binding.result()
    tmp = LIB.with_suffix(".so.tmp")
    subprocess.run([nvcc, *ARCH, "-shared", *[str(o) for o in objs], "-o", str(tmp)], check=True)
    os.replace(tmp, LIB)
    run(bind_link, BIND.name)
    os.replace(str(BIND) + ".tmp", BIND)
    return LIB


if __name__ == "__main__":
    build_library(force="--force" in sys.argv, verbose="-v" in sys.argv)
    print(LIB)
