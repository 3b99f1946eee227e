"""Build the sm_100a shared library ``_fnx.so`` in-tree with nvcc, and the native Python
binding of the verify-step operators ``_fnx_ops.so`` (csrc/binding.cpp) with g++ and torch's headers.

    python -m flash_next_rtxpro6000_b200.build [--force]

Each ``csrc/*.cu`` file is compiled to an object in parallel, then linked into one
shared library with the CUDA runtime linked statically (the library then depends only on
the driver, not on a particular libcudart).  The binding links that library (found beside it)
and torch.
"""

from __future__ import annotations

import argparse
import os
import shutil
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

PKG = Path(__file__).resolve().parent
CSRC = PKG / "csrc"
INCLUDE = PKG.parent / "include"
LIB_PATH = PKG / "_fnx.so"
OPS_PATH = PKG / "_fnx_ops.so"
OBJ_DIR = PKG / "_build"

SOURCES = ["fnx_api.cu", "dense_gemv.cu", "dense_gemv_slice.cu", "dense_gemv_norm.cu", "dense_tc.cu",
           "moe_gemv.cu",
           "moe_fused.cu", "moe_lean.cu", "nvfp4_codec.cu", "router.cu", "topk1.cu",
           "rotary.cu", "tree_attn.cu", "tree_attn_tc.cu", "sample.cu", "sample_many.cu",
           "token_probs.cu", "token_probs_many.cu",
           "append8.cu", "tree_attn8.cu", "tree_attn8_tc.cu", "verify.cu", "compact.cu"]
BINDING = "binding.cpp"
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
FLAGS = ["-O3", "-lineinfo", "-std=c++17", "--expt-relaxed-constexpr", "-Xcompiler", "-fPIC",
         "-I" + str(INCLUDE)]


def nvcc() -> str:
    cand = os.environ.get("NVCC") or shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not Path(cand).exists():
        raise RuntimeError("nvcc not found: the sm_100a library cannot be built")
    return cand


def _newer(path: Path, inputs) -> bool:
    return path.exists() and all(p.stat().st_mtime <= path.stat().st_mtime for p in inputs)


def library_up_to_date() -> bool:
    return _newer(LIB_PATH, [CSRC / s for s in SOURCES] + sorted(CSRC.glob("*.cuh")) + sorted(CSRC.glob("*.h")) +
                  sorted(INCLUDE.glob("*.h")))


def binding_build() -> str:
    """What a binding is made for: torch's C++ interface changes from build to build, the
    interpreter's from version to version."""
    import sysconfig

    import torch

    return (f"fnx binding for torch {torch.__version__} abi {int(torch._C._GLIBCXX_USE_CXX11_ABI)} "
            f"python {sysconfig.get_config_var('SOABI')};")


def binding_fits() -> bool:
    """Whether ``_fnx_ops.so`` is there and was made for this torch and interpreter (it holds the text)."""
    return OPS_PATH.exists() and binding_build().encode() in OPS_PATH.read_bytes()


def up_to_date() -> bool:
    return library_up_to_date() and binding_fits() and \
        _newer(OPS_PATH, [CSRC / BINDING] + sorted(INCLUDE.glob("*.h")))


def build(force: bool = False, verbose: bool = False) -> Path:
    """Compile the library and the binding if any of their sources is newer; returns the library's path."""
    if force or not up_to_date():
        build_library(force, verbose)
        build_binding()
    return LIB_PATH


def build_library(force: bool = False, verbose: bool = False) -> Path:
    """Compile the library if any source is newer than it; returns its path."""
    if not force and library_up_to_date():
        return LIB_PATH
    OBJ_DIR.mkdir(exist_ok=True)
    cc = nvcc()
    extra = ["-Xptxas", "-v"] if verbose else []

    def compile_one(src: str) -> Path:
        obj = OBJ_DIR / (Path(src).stem + ".o")
        cmd = [cc, *ARCH, *FLAGS, *extra, "-c", str(CSRC / src), "-o", str(obj)]
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"nvcc failed on {src}:\n{r.stdout}\n{r.stderr}")
        if verbose:
            sys.stderr.write(r.stderr)
        return obj

    with ThreadPoolExecutor(max_workers=len(SOURCES)) as ex:
        objs = list(ex.map(compile_one, SOURCES))
    tmp = LIB_PATH.with_suffix(".so.tmp")
    cmd = [cc, *ARCH, "-shared", "-cudart", "static", "-o", str(tmp), *map(str, objs)]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"link failed:\n{r.stdout}\n{r.stderr}")
    os.replace(tmp, LIB_PATH)
    return LIB_PATH


def build_binding() -> Path:
    """Compile csrc/binding.cpp against the interpreter's torch, linked to ``_fnx.so``."""
    import sysconfig

    import torch

    root = Path(torch.__file__).resolve().parent
    cuda = Path(nvcc()).resolve().parent.parent
    tmp = OPS_PATH.with_suffix(".so.tmp")
    cmd = [os.environ.get("CXX") or "g++", "-O2", "-std=c++17", "-fPIC", "-shared",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
           f'-DFNX_BINDING_BUILD="{binding_build()}"',
           f"-I{root}/include", f"-I{root}/include/torch/csrc/api/include",
           f"-I{sysconfig.get_paths()['include']}", f"-I{cuda}/include", str(CSRC / BINDING),
           "-o", str(tmp), f"-L{PKG}", "-l:_fnx.so", f"-L{root}/lib", "-lc10", "-lc10_cuda", "-ltorch",
           "-ltorch_cpu", "-ltorch_python", "-Wl,-rpath,$ORIGIN"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"g++ failed on {BINDING}:\n{r.stdout}\n{r.stderr}")
    os.replace(tmp, OPS_PATH)
    return OPS_PATH


def main():
    ap = argparse.ArgumentParser()
    ap.add_argument("--force", action="store_true")
    ap.add_argument("--verbose", action="store_true")
    a = ap.parse_args()
    print(build(force=a.force, verbose=a.verbose))


if __name__ == "__main__":
    main()
