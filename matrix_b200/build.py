"""Builds libmtxc.so (the C-ABI backend) in-tree for sm_100a.

Run as ``python -m matrix_b200.build`` (or through ``__graft_entry__.build()``).  nvcc
cross-compiles without a GPU.  Objects go to ``matrix_b200/_build/``; the library to
``matrix_b200/lib/libmtxc.so``, which travels with the source tree to the GPU box.  The
CUDA runtime is linked statically so the library does not depend on which libcudart the
host process (e.g. PyTorch) loaded.  ``binding/`` is compiled against the installed torch into the Python
module ``lib/_lm.so``, and again when another torch is installed; where there is none with CUDA it is left out.
"""
from __future__ import annotations

import concurrent.futures as cf
import os
import shutil
import subprocess
import sys
import sysconfig
from pathlib import Path

PKG = Path(__file__).resolve().parent
REPO = PKG.parent
CSRC = PKG / "csrc"
BUILD = PKG / "_build"
LIBDIR = PKG / "lib"
LIB = LIBDIR / "libmtxc.so"
HOST = PKG / "host"
HOST_LIB = LIBDIR / "libmtx.so"
BINDING = PKG / "binding"
BINDING_LIB = LIBDIR / "_lm.so"
BINDING_TORCH = BUILD / "_lm.torch"  # the torch that BINDING_LIB was compiled against
INCLUDE = REPO / "include"

ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
NVCC_FLAGS = ["-O3", "-std=c++17", "-lineinfo", "-Xcompiler", "-fPIC", "-Xcompiler", "-Wall",
              "--expt-relaxed-constexpr", "-I", str(INCLUDE), "-I", str(CSRC)]
CXX_FLAGS = ["-O2", "-std=c++17", "-fPIC", "-Wall", "-I", str(INCLUDE)]


def nvcc() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and Path(cand).exists():
            return cand
    raise RuntimeError("nvcc not found")


def _stale(obj: Path, deps: list[Path]) -> bool:
    if not obj.exists():
        return True
    t = obj.stat().st_mtime
    return any(d.stat().st_mtime > t for d in deps)


def _run(cmd: list[str], verbose: bool = False) -> str:
    if verbose:
        print(" ".join(cmd), file=sys.stderr)
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"compile failed: {' '.join(cmd)}\n{res.stdout}\n{res.stderr}")
    return res.stdout + res.stderr


def build_binding(headers: list[Path], verbose: bool = False) -> Path | None:
    """Compiles the Python module over torch tensors; None, with a message, where there is no torch with CUDA."""
    try:
        import torch
    except (ImportError, OSError) as e:
        missing = f"torch cannot be imported: {e}"
    else:
        missing = "" if torch.version.cuda else f"torch {torch.__version__} is built without CUDA"
    if missing:
        print(f"{BINDING_LIB.name} left out ({missing}); the C ABI does not need it", file=sys.stderr)
        return None
    torch_dir = Path(torch.__file__).resolve().parent
    against = f"{torch.__version__} {torch_dir}"
    srcs = sorted(BINDING.glob("*.cpp"))
    if _stale(BINDING_LIB, [*srcs, LIB, *headers]) or not BINDING_TORCH.exists() or BINDING_TORCH.read_text() != against:
        cuda_include = Path(nvcc()).resolve().parent.parent / "include"
        _run(["g++", *CXX_FLAGS, "-shared", "-I", str(torch_dir / "include"),
              "-I", str(torch_dir / "include" / "torch" / "csrc" / "api" / "include"),
              "-I", sysconfig.get_paths()["include"], "-I", str(cuda_include),
              f"-D_GLIBCXX_USE_CXX11_ABI={int(torch.compiled_with_cxx11_abi())}",
              f'-DMTX_TORCH_VERSION="{torch.__version__}"', "-o", str(BINDING_LIB), *map(str, srcs), "-L", str(LIBDIR),
              "-lmtxc", "-L", str(torch_dir / "lib"), "-ltorch_python", "-ltorch_cuda", "-ltorch_cpu", "-ltorch",
              "-lc10_cuda", "-lc10", "-Wl,-rpath,$ORIGIN"], verbose)
        BINDING_TORCH.write_text(against)
    return BINDING_LIB


def build(verbose: bool = False, ptxas_info: bool = False) -> Path:
    BUILD.mkdir(exist_ok=True)
    LIBDIR.mkdir(exist_ok=True)
    headers = sorted(CSRC.glob("*.cuh")) + sorted(CSRC.glob("*.h")) + sorted(INCLUDE.glob("*.h"))
    jobs = []
    objs = []
    for src in sorted(CSRC.glob("*.cu")):
        obj = BUILD / (src.stem + ".o")
        objs.append(obj)
        if _stale(obj, [src, *headers]) or ptxas_info:
            cmd = [nvcc(), *ARCH, *NVCC_FLAGS, "-c", str(src), "-o", str(obj)]
            if ptxas_info:
                cmd[1:1] = ["-Xptxas", "-v"]
            jobs.append(cmd)
    for src in sorted(CSRC.glob("*.cpp")):
        obj = BUILD / (src.stem + ".o")
        objs.append(obj)
        if _stale(obj, [src, *headers]):
            jobs.append(["g++", *CXX_FLAGS, "-c", str(src), "-o", str(obj)])

    def run(cmd: list[str]) -> str:
        return _run(cmd, verbose)

    with cf.ThreadPoolExecutor(max_workers=max(1, min(len(jobs), os.cpu_count() or 4))) as ex:
        for out in ex.map(run, jobs):
            if out.strip() and (verbose or ptxas_info):
                print(out, file=sys.stderr)
    if jobs or not LIB.exists() or _stale(LIB, objs):
        run([nvcc(), *ARCH, "-shared", "-cudart", "static", "-o", str(LIB), *map(str, objs), "-ldl"])
    # the C++ host mirror of the reference API (mtx.hpp), a plain C++ library over the C ABI
    host_srcs = sorted(HOST.glob("*.cpp"))
    if host_srcs and (not HOST_LIB.exists() or _stale(HOST_LIB, [*host_srcs, *HOST.glob("*.hpp"), LIB, *headers])):
        cuda_include = Path(nvcc()).resolve().parent.parent / "include"  # NVTX v3 (header-only)
        run(["g++", "-O2", "-std=c++17", "-fPIC", "-Wall", "-shared", "-I", str(INCLUDE), "-I", str(HOST),
             "-I", str(cuda_include), "-o", str(HOST_LIB), *map(str, host_srcs), "-L", str(LIBDIR), "-lmtxc",
             "-ldl", "-Wl,-rpath,$ORIGIN"])
    build_binding(headers, verbose)
    return LIB


if __name__ == "__main__":
    build(verbose="-v" in sys.argv, ptxas_info="--ptxas-info" in sys.argv)
    print(LIB)
