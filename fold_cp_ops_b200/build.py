"""Ahead-of-time build of ``libtrimul_sm100.so`` with nvcc for sm_100a, and of the host module ``_pair_host.so``.

Both are built in-tree (next to this file) so that they travel with a snapshot of the repository; there is no JIT.  The
library holds every kernel and knows nothing of torch; the host module (argument checks, allocation and gradients of
the pair-stream operators, C++ against torch's headers) holds no kernel and calls the library.  ``python -m
fold_cp_ops_b200.build`` rebuilds it; :func:`ensure_built` rebuilds only when a source is newer
than the library.
"""
from __future__ import annotations

import os
import shutil
import subprocess
import sys
from pathlib import Path

PKG_DIR = Path(__file__).resolve().parent
CSRC = PKG_DIR / "csrc"
LIB_PATH = PKG_DIR / "libtrimul_sm100.so"

SOURCES = ("trimul_capi.cu", "ln_gated_proj.cu", "tri_contract.cu", "tri_contract_pair.cu", "ln_out_proj.cu", "peer_sync.cu",
           "forward_static.cu", "pair_norm.cu", "pair_norm_grad.cu", "pair_embed.cu")
HEADERS = ("sm100_ptx.cuh", "trimul_common.cuh", "trimul_kernels.h", "tri_contract_epilogue.cuh", "pair_stream.cuh")
PUBLIC_HEADERS = ("trimul_sm100.h", "pair_stream_sm100.h")
HOST_SOURCE = "pair_host.cpp"
HOST_PATH = PKG_DIR / "_pair_host.so"

NVCC_FLAGS = (
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-lineinfo", "-O3", "-std=c++17",
    "-Xcompiler", "-fPIC", "-shared",
    "--use_fast_math",
    "--threads", "0",
    "-diag-suppress", "177",
)


def source_digest() -> str:
    """sha256 over the CUDA sources, their headers and the public header, in a fixed order.  Compiled into
    the library (``trimul_sm100_build_id``) so that the loader can tell a library built from other sources
    without relying on file times, which a copy of the tree does not preserve."""
    import hashlib

    h = hashlib.sha256()
    for f in [CSRC / s for s in SOURCES + HEADERS + (HOST_SOURCE,)] + [PKG_DIR.parent / "include" / h for h in PUBLIC_HEADERS]:
        h.update(f.name.encode())
        h.update(f.read_bytes())
    return h.hexdigest()[:32]


def _nvcc() -> str:
    cand = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not Path(cand).exists():
        raise RuntimeError("nvcc not found; libtrimul_sm100.so cannot be built")
    return cand


def is_stale() -> bool:
    if not LIB_PATH.exists() or not HOST_PATH.exists():
        return True
    t = min(LIB_PATH.stat().st_mtime, HOST_PATH.stat().st_mtime)
    deps = [CSRC / s for s in SOURCES + HEADERS + (HOST_SOURCE,)] + [PKG_DIR.parent / "include" / h for h in PUBLIC_HEADERS]
    return any(d.exists() and d.stat().st_mtime > t for d in deps)


def build(verbose: bool = False, ptxas_info: bool = False, ablate: int = 0) -> Path:
    """Compile every kernel for sm_100a into one shared library, and the host module; returns the library's path.

    ``ablate`` != 0 builds a PROFILING library ``libtrimul_sm100_ablate<bits>.so`` beside the real one, in
    which roles of the projection kernel do no work (``TRIMUL_ABLATE`` in ``csrc/ln_gated_proj.cu``); select
    it with ``CPO_TRIMUL_LIB``.  Its results are wrong by construction; it only exists to be timed."""
    srcs = [str(CSRC / s) for s in SOURCES if (CSRC / s).exists()]
    out = LIB_PATH if not ablate else PKG_DIR / f"libtrimul_sm100_ablate{int(ablate)}.so"
    extra = [f"-DTRIMUL_ABLATE={int(ablate)}"] if ablate else []
    extra.append(f'-DTRIMUL_BUILD_ID="{source_digest()}"')
    cmd = [_nvcc(), *NVCC_FLAGS, *extra, *(["-Xptxas", "-v"] if ptxas_info else []), "-o", str(out), *srcs]
    if verbose:
        print(" ".join(cmd), file=sys.stderr)
    proc = subprocess.run(cmd, capture_output=True, text=True)
    if proc.returncode != 0:
        raise RuntimeError(f"nvcc failed ({proc.returncode}):\n{proc.stdout}\n{proc.stderr}")
    if verbose or ptxas_info:
        sys.stderr.write(proc.stderr)
    if not ablate:
        _build_host(verbose)
    return out


def _build_host(verbose: bool = False) -> Path:
    """Compile the host module against the installed torch."""
    import sysconfig

    import torch

    cxx = shutil.which("g++")
    if cxx is None:
        raise RuntimeError("g++ not found; _pair_host.so cannot be built")
    root = Path(torch.__file__).parent
    cuda = Path(_nvcc()).resolve().parent.parent
    include = (root / "include", root / "include" / "torch" / "csrc" / "api" / "include", cuda / "include",
               Path(sysconfig.get_paths()["include"]))
    cmd = [cxx, "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden", "-DTORCH_EXTENSION_NAME=_pair_host",
           "-DTORCH_API_INCLUDE_EXTENSION_H", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch.compiled_with_cxx11_abi())}",
           f'-DTRIMUL_BUILD_ID="{source_digest()}"', *(a for p in include for a in ("-isystem", str(p))),
           str(CSRC / HOST_SOURCE), "-o", str(HOST_PATH), f"-L{root / 'lib'}", "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch",
           "-ltorch_python"]
    if verbose:
        print(" ".join(cmd), file=sys.stderr)
    proc = subprocess.run(cmd, capture_output=True, text=True)
    if proc.returncode != 0:
        raise RuntimeError(f"g++ failed ({proc.returncode}):\n{proc.stdout}\n{proc.stderr}")
    return HOST_PATH


def ensure_built() -> Path:
    if is_stale():
        build()
    return LIB_PATH


if __name__ == "__main__":
    bits = int(sys.argv[sys.argv.index("--ablate") + 1]) if "--ablate" in sys.argv else 0
    print(build(verbose=True, ptxas_info="--ptxas" in sys.argv, ablate=bits))
