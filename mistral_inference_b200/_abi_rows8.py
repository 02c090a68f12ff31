"""ctypes binding of libmb200_rows8.so (C ABI: include/mistral_b200_rows8.h): Linears of 8-bit numbers.

Same rules as `_abi`: the only place Python touches this library, and no fallback -- a missing library is built once
in-tree by `build.build_rows8()` (a fresh checkout has no binaries), a failing call raises.
"""
import ctypes
import functools
from ctypes import c_char_p, c_float, c_int, c_int64, c_void_p
from typing import Optional

import torch

from . import build
from ._abi import Mb200Error, _stream

ABI_VERSION = 1
BLOCK = 128     # numbers that share a scale
MAX_ROWS = 1 << 24
MAX_NORM = 65536
_lib: Optional[ctypes.CDLL] = None

P, I = c_void_p, c_int64
_SIGNATURES = {
    "mb8_abi_version": (c_int, []),
    "mb8_last_error": (c_char_p, []),
    "mb8_quantise": (c_int, [P, I, c_int, P, P, I, I, P]),
    "mb8_norm": (c_int, [P, I, P, I, P, c_int, P, P, P, I, I, c_float, P]),
    "mb8_rotate": (c_int, [P, P, P, P, P, P, P, I, I, I, P]),
    "mb8_product_scratch": (I, [I, I, I]),
    "mb8_multiply": (c_int, [P, P, P, P, P, I, c_int, I, I, I, c_int, P, I, P]),
    "mb8_gate": (c_int, [P, P, P, P, P, P, I, I, I, c_int, P, I, P]),
}


def lib() -> ctypes.CDLL:
    global _lib
    if _lib is None:
        handle = ctypes.CDLL(str(build.build_rows8()))
        for name, (restype, argtypes) in _SIGNATURES.items():
            fn = getattr(handle, name)
            fn.restype, fn.argtypes = restype, argtypes
        if handle.mb8_abi_version() != ABI_VERSION:
            raise Mb200Error(f"libmb200_rows8 ABI {handle.mb8_abi_version()} != expected {ABI_VERSION}")
        _lib = handle
    return _lib


_lazy = {}  # name -> entry point, once the library is loaded


def call(name: str, device: int, *args) -> None:
    """The entry point on the current stream of `device`, whatever the current device is."""
    fn = _lazy.get(name)
    if fn is None:
        fn = _lazy[name] = getattr(lib(), name)
    if device == torch._C._cuda_getDevice():
        rc = fn(*args, _stream())
    else:
        with torch.cuda.device(device):
            rc = fn(*args, _stream())
    if rc != 0:
        msg = lib().mb8_last_error()
        raise Mb200Error(f"{name} failed ({rc}): {msg.decode() if msg else '?'}")


@functools.lru_cache(maxsize=256)
def _scratch_bytes(device: int, T: int, N: int, K: int) -> int:
    """How a product is cut goes by its device's SMs: the same device is asked that the call will run on."""
    with torch.cuda.device(device):
        return lib().mb8_product_scratch(T, N, K)


STREAM_TOKENS = 128  # up to so many tokens a product needs no scratch


def product(name: str, device: int, x, w, out: tuple, T: int, N: int, n: int) -> None:
    """mb8_multiply or mb8_gate of x [T, K] and w [N, K]; n: what the entry point counts its results by."""
    need = _scratch_bytes(device, T, N, x.cols) if T > STREAM_TOKENS else 0
    scratch = x.codes.new_empty(need) if need else None
    call(name, device, x.codes.data_ptr(), x.scales.data_ptr(), w.codes.data_ptr(), w.scales.data_ptr(), *out, T, n, x.cols, w.fixed, None if scratch is None else scratch.data_ptr(), need)


def rotate(qkv, rope, positions, rows, q, k, v, n_heads: int, n_kv_heads: int) -> None:
    """Behind the model's own product: tensors as the model makes them, contiguous and of one device."""
    for t in (qkv, rope, positions, q, k, v):
        assert t.get_device() == qkv.get_device() and t.is_contiguous(), "contiguous tensors of one device"
    assert rows is None or (rows.get_device() == qkv.get_device() and rows.is_contiguous())
    call("mb8_rotate", qkv.get_device(), qkv.data_ptr(), rope.data_ptr(), positions.data_ptr(), None if rows is None else rows.data_ptr(), q.data_ptr(), k.data_ptr(), v.data_ptr(), qkv.shape[0],
         n_heads, n_kv_heads)
