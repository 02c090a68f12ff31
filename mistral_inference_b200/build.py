"""Builds libmb200.so (the C-ABI CUDA library) in-tree with nvcc for sm_100a.

In-tree, so that a copy of the checkout carries its built libraries with it (a JIT cache would not).
`python -m mistral_inference_b200.build [--force] [--verbose]`
"""
import hashlib
import os
import subprocess
import sys
from pathlib import Path

PKG = Path(__file__).resolve().parent
CSRC = PKG / "csrc"
LIB = PKG / "libmb200.so"
STAMP = PKG / "csrc" / ".build_stamp"

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-O3", "-std=c++17", "-lineinfo",
    "-Xcompiler", "-fPIC", "-shared",
    "--expt-relaxed-constexpr",
]


def _extra_defines():
    return [f"-D{d}" for d in os.environ.get("MB200_DEFINES", "").split() if d]


def _sources_digest() -> str:
    h = hashlib.sha256()
    for f in sorted(list(CSRC.glob("*.cu")) + list(CSRC.glob("*.cuh")) + [PKG.parent / "include" / "mistral_b200.h"]):
        h.update(f.name.encode())
        h.update(f.read_bytes())
    h.update(" ".join(NVCC_FLAGS + _extra_defines()).encode())
    return h.hexdigest()


def build_variant(name: str, defines) -> Path:
    """An extra in-tree library with additional -D flags (A/B experiments: MB200_LIB_PATH selects it at run time)."""
    out = PKG / f"libmb200_{name}.so"
    nvcc = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")
    cmd = [nvcc, *NVCC_FLAGS, *[f"-D{d}" for d in defines], "-o", str(out)] + [str(f) for f in sorted(CSRC.glob("*.cu"))]
    proc = subprocess.run(cmd, capture_output=True, text=True)
    if proc.returncode != 0:
        sys.stderr.write(proc.stdout + proc.stderr)
        raise RuntimeError(f"nvcc failed ({proc.returncode})")
    return out


def build_library(force: bool = False, verbose: bool = False) -> Path:
    digest = _sources_digest()
    if not force and LIB.exists() and STAMP.exists() and STAMP.read_text().strip() == digest:
        return LIB
    nvcc = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")
    cmd = [nvcc, *NVCC_FLAGS, *_extra_defines(), "-Xptxas", "-v", "-o", str(LIB)] + [str(f) for f in sorted(CSRC.glob("*.cu"))]
    proc = subprocess.run(cmd, capture_output=True, text=True)
    (CSRC / "ptxas.log").write_text(proc.stderr)
    if proc.returncode != 0:
        sys.stderr.write(proc.stdout + proc.stderr)
        raise RuntimeError(f"nvcc failed ({proc.returncode}): {' '.join(cmd)}")
    if verbose:
        print(proc.stderr)
    STAMP.write_text(digest)
    return LIB


def _build_small(src: Path, lib: Path, others, flags=(), force: bool = False) -> Path:
    """A library of its own of the sources in `src` (and of `others`, which they include), so that who needs only it compiles only them (seconds).  Safe when several
    processes start at once: the output is written under a private name and renamed."""
    sources = sorted(src.glob("*.cu"))
    h = hashlib.sha256()
    for f in sources + sorted(src.glob("*.cuh")) + sorted(src.glob("*.h")) + list(others):
        h.update(f.name.encode())
        h.update(f.read_bytes())
    h.update(" ".join(NVCC_FLAGS).encode())
    digest = h.hexdigest()
    stamp = src / ".build_stamp"
    if not force and lib.exists() and stamp.exists() and stamp.read_text().strip() == digest:
        return lib
    nvcc = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")
    tmp = PKG / f".{lib.stem}.{os.getpid()}.so"
    cmd = [nvcc, *NVCC_FLAGS, *flags, "-o", str(tmp)] + [str(f) for f in sources]
    proc = subprocess.run(cmd, capture_output=True, text=True)
    if proc.returncode != 0:
        sys.stderr.write(proc.stdout + proc.stderr)
        raise RuntimeError(f"nvcc failed ({proc.returncode}): {' '.join(cmd)}")
    os.replace(tmp, lib)
    stamp.write_text(digest)
    return lib


INCLUDE = PKG.parent / "include"
HYBRID_SRC = CSRC / "hybrid"
HYBRID_LIB = PKG / "libmb200_hybrid.so"


def build_hybrid(force: bool = False) -> Path:
    """libmb200_hybrid.so: the kernels of layered decoders (csrc/hybrid/)."""
    return _build_small(HYBRID_SRC, HYBRID_LIB, [CSRC / "stream_linear.cuh", CSRC / "device_info.cuh"] + sorted(INCLUDE.glob("mistral_b200_hybrid*.h")), ("--threads", "0"), force)


PAGED_SRC = CSRC / "paged"
PAGED_LIB = PKG / "libmb200_paged.so"


def build_paged(force: bool = False) -> Path:
    """libmb200_paged.so: pages of 8-bit keys and values and the scores of tokens (csrc/paged/)."""
    headers = ["common.cuh", "device_info.cuh", "epilogue.cuh", "sigmoid.cuh", "gemm_tcgen05.cuh", "gemm_mma.cuh", "split_schedule.cuh", "decode_megakernel.cuh", "attn_decode.cuh",
               "attn_prompt_tcgen05.cuh"]
    return _build_small(PAGED_SRC, PAGED_LIB, [CSRC / h for h in headers] + [INCLUDE / h for h in ("mistral_b200.h", "mistral_b200_paged.h")], force=force)


if __name__ == "__main__":
    print(build_paged(force="--force" in sys.argv))
    print(build_hybrid(force="--force" in sys.argv))
    print(build_library(force="--force" in sys.argv, verbose="--verbose" in sys.argv))
