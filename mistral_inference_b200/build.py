"""Builds libmb200.so (the C-ABI CUDA library) in-tree with nvcc for sm_100a.

In-tree, so that a copy of the checkout carries its built libraries with it (a JIT cache would not).
`python -m mistral_inference_b200.build [--force] [--verbose]`
"""
import hashlib
import os
import re
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


_INCLUDE = re.compile(r'^\s*#\s*include\s+"([^"]+)"', re.M)


def _with_included(sources) -> list:
    """The sources and all files of the checkout that they include."""
    found = todo = {f.resolve() for f in sources}
    while todo:
        todo = {f for p in todo for f in ((p.parent / name).resolve() for name in _INCLUDE.findall(p.read_text())) if f.exists()} - found
        found = found | todo
    return sorted(found)


def _build_small(src: Path, lib: Path, flags=(), force: bool = False) -> Path:
    """A library of its own of the sources in `src` (and of what they include), so that who needs only it compiles only them (seconds).  Safe when several
    processes start at once: the output is written under a private name and renamed."""
    sources = sorted(src.glob("*.cu"))
    h = hashlib.sha256()
    for f in _with_included(sources):
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


HYBRID_SRC = CSRC / "hybrid"
HYBRID_LIB = PKG / "libmb200_hybrid.so"


def build_hybrid(force: bool = False) -> Path:
    """libmb200_hybrid.so: the kernels of layered decoders (csrc/hybrid/)."""
    return _build_small(HYBRID_SRC, HYBRID_LIB, ("--threads", "0"), force)


PAGED_SRC = CSRC / "paged"
PAGED_LIB = PKG / "libmb200_paged.so"


def build_paged(force: bool = False) -> Path:
    """libmb200_paged.so: pages of 8-bit keys and values and the scores of tokens (csrc/paged/)."""
    return _build_small(PAGED_SRC, PAGED_LIB, force=force)


ROWS8_SRC = CSRC / "rows8"
ROWS8_LIB = PKG / "libmb200_rows8.so"


def build_rows8(force: bool = False) -> Path:
    """libmb200_rows8.so: Linears of 8-bit numbers (csrc/rows8/)."""
    return _build_small(ROWS8_SRC, ROWS8_LIB, force=force)


ROWS8_HOST = PKG / "mb200_rows8_host.so"


def build_rows8_host(force: bool = False) -> Path:
    """mb200_rows8_host.so: the Python extension behind rows8.py (csrc/rows8/rows8_host.cpp, some 10 s), against the torch and the Python that run this."""
    import sysconfig

    import torch

    src, stamp = ROWS8_SRC / "rows8_host.cpp", ROWS8_SRC / ".build_stamp_host"
    top = Path(torch.__file__).resolve().parent
    flags = ["-O2", "-std=c++17", "-shared", "-fPIC", "-fvisibility=hidden", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}"]
    includes = [str(top / "include"), str(top / "include" / "torch" / "csrc" / "api" / "include"), sysconfig.get_paths()["include"], "/usr/local/cuda/include"]
    h = hashlib.sha256()
    for f in _with_included([src]):
        h.update(f.read_bytes())
    h.update(" ".join(flags + [torch.__version__, sys.version]).encode())
    digest = h.hexdigest()
    if not force and ROWS8_HOST.exists() and stamp.exists() and stamp.read_text().strip() == digest:
        return ROWS8_HOST
    tmp = PKG / f".{ROWS8_HOST.stem}.{os.getpid()}.so"
    cmd = [os.environ.get("CXX", "g++"), *flags, *[f"-I{d}" for d in includes], "-o", str(tmp), str(src), f"-L{top / 'lib'}", "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch_cuda", "-ltorch_python"]
    proc = subprocess.run(cmd, capture_output=True, text=True)
    if proc.returncode != 0:
        sys.stderr.write(proc.stdout + proc.stderr)
        raise RuntimeError(f"g++ failed ({proc.returncode}): {' '.join(cmd)}")
    os.replace(tmp, ROWS8_HOST)
    stamp.write_text(digest)
    return ROWS8_HOST


if __name__ == "__main__":
    print(build_rows8(force="--force" in sys.argv))
    print(build_rows8_host(force="--force" in sys.argv))
    print(build_paged(force="--force" in sys.argv))
    print(build_hybrid(force="--force" in sys.argv))
    print(build_library(force="--force" in sys.argv, verbose="--verbose" in sys.argv))
