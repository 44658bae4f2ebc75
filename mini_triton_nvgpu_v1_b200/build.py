"""Builds the in-tree shared library ``libtbgemm.so`` (the C ABI of
``include/tb_gemm.h``) with nvcc for sm_100a, and ``_tbtorch.so`` (the calls of
``grouped.py`` on torch tensors) with g++ against torch's headers.

Both are written next to this file so they travel with the source tree;
``python -m mini_triton_nvgpu_v1_b200.build`` rebuilds them. Without torch only
the C library is built.
"""
from __future__ import annotations

import os
import shutil
import subprocess
import sys
from pathlib import Path

PKG = Path(__file__).resolve().parent
ROOT = PKG.parent
CSRC = PKG / "csrc"
LIB = PKG / "libtbgemm.so"
TORCH_LIB = PKG / "_tbtorch.so"
TORCH_TAG = PKG / "_tbtorch.so.tag"  # the torch and Python that it was built against

SOURCES = ["tb_plan.cpp", "tb_dynamic.cpp", "tb_shard.cpp", "tb_launch.cu", "tb_grouped.cu", "tb_quantize.cu", "tb_peer.cu", "tb_nccl.cpp"]
HEADERS = ["tb_plan.h", "tb_mapping.h", "tb_sm100.cuh", "tb_wait.cuh"]

ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]


def nvcc() -> str:
    cand = os.environ.get("NVCC") or shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    return cand


def _stale(out: Path, inputs: list[Path]) -> bool:
    if not out.exists():
        return True
    t = out.stat().st_mtime
    return any(p.stat().st_mtime > t for p in inputs)


def _run(cmd: list[str], verbose: bool) -> str:
    if verbose:
        print(" ".join(cmd), file=sys.stderr)
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"{Path(cmd[0]).name} failed ({r.returncode}):\n{r.stdout}\n{r.stderr}")
    return r.stdout + r.stderr


def build_torch(force: bool = False, verbose: bool = False) -> Path | None:
    """``_tbtorch.so``, or None where there is no torch: it is only looked up
    here, not imported. Built anew for another torch or Python."""
    import importlib.util
    import sysconfig
    src = CSRC / "tb_torch.cpp"
    spec = importlib.util.find_spec("torch")
    if spec is None or spec.origin is None:
        print("torch is not installed: _tbtorch.so, the calls of grouped.py on its tensors, is left out",
              file=sys.stderr)
        return None
    torch = Path(spec.origin).parent
    version = torch / "version.py"
    tag = f"{sysconfig.get_config_var('SOABI')}\n{torch}\n{version.read_text() if version.exists() else ''}"
    if (not force and not _stale(TORCH_LIB, [src, ROOT / "include" / "tb_gemm.h", Path(__file__)])
            and TORCH_TAG.exists() and TORCH_TAG.read_text() == tag):
        return TORCH_LIB
    cuda = Path(nvcc()).resolve().parents[1]
    tmp = TORCH_LIB.with_suffix(".so.tmp")
    _run([os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-fPIC", "-shared", "-Wall", "-Wno-unknown-pragmas",
          "-I", sysconfig.get_paths()["include"], "-I", str(torch / "include"),
          "-I", str(torch / "include" / "torch" / "csrc" / "api" / "include"), "-I", str(cuda / "include"),
          str(src), "-o", str(tmp), "-L", str(torch / "lib"), "-ltorch_python", "-ltorch_cpu", "-lc10", "-lc10_cuda"],
         verbose)
    os.replace(tmp, TORCH_LIB)
    TORCH_TAG.write_text(tag)
    return TORCH_LIB


def build(force: bool = False, verbose: bool = False, ptxas_v: bool = False) -> Path:
    """Compiles each source to an object (in parallel, under ``_build/``) and
    links ``libtbgemm.so``; skipped when the library is newer than every input.
    Then ``_tbtorch.so``, where there is a torch."""
    _build_library(force, verbose, ptxas_v)
    build_torch(force, verbose)
    return LIB


def _build_library(force: bool, verbose: bool, ptxas_v: bool) -> None:
    inputs = [CSRC / s for s in SOURCES] + [CSRC / h for h in HEADERS] + [ROOT / "include" / "tb_gemm.h",
                                                                           Path(__file__)]
    if not force and not _stale(LIB, inputs):
        return
    objdir = ROOT / "_build"
    objdir.mkdir(exist_ok=True)
    common = [nvcc(), *ARCH, "-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC",
              "-Xcompiler", "-Wall", "--expt-relaxed-constexpr",
              "-I", str(ROOT / "include"), "-I", str(CSRC)]
    objs = [objdir / (s + ".o") for s in SOURCES]
    from concurrent.futures import ThreadPoolExecutor
    with ThreadPoolExecutor(max_workers=len(SOURCES)) as ex:
        outs = list(ex.map(lambda so: _run(common + (["-Xptxas", "-v"] if ptxas_v and so[0].endswith(".cu")
                                                     else []) + ["-c", str(CSRC / so[0]), "-o", str(so[1])],
                                           verbose), zip(SOURCES, objs)))
    tmp = LIB.with_suffix(".so.tmp")
    _run([nvcc(), *ARCH, "-shared", *[str(o) for o in objs], "-o", str(tmp), "-ldl"], verbose)
    if verbose or ptxas_v:
        print("".join(outs), file=sys.stderr)
    os.replace(tmp, LIB)


if __name__ == "__main__":
    build(force="--force" in sys.argv, verbose=True, ptxas_v="--ptxas-v" in sys.argv)
    print(LIB)
