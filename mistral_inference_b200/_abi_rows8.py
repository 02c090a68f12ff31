"""ctypes binding of libmb200_rows8.so (C ABI: include/mistral_b200_rows8.h): Linears of 8-bit numbers.

Same rules as `_abi`: the only place Python touches this library, and no fallback -- a missing library is built once
in-tree by `build.build_rows8()` (a fresh checkout has no binaries), a failing call raises.  The operators of rows8.py go
through a Python extension over the same C ABI (`host()`), which does in C++ what a call needs from the host.
"""
import ctypes
import importlib.util
from ctypes import c_char_p, c_float, c_int, c_int64, c_void_p
from importlib.machinery import ExtensionFileLoader
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


_host = None


def host():
    """The extension (csrc/rows8/rows8_host.cpp), bound to the library's entry points."""
    global _host
    if _host is None:
        handle, path = lib(), str(build.build_rows8_host())
        loader = ExtensionFileLoader("mb200_rows8_host", path)
        module = importlib.util.module_from_spec(importlib.util.spec_from_file_location("mb200_rows8_host", path, loader=loader))
        loader.exec_module(module)
        entries = ("mb8_last_error", "mb8_quantise", "mb8_norm", "mb8_multiply", "mb8_gate", "mb8_product_scratch")
        module.bind(Mb200Error, *[ctypes.cast(getattr(handle, n), c_void_p).value for n in entries])
        _host = module
    return _host


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


def rotate(qkv, rope, positions, rows, q, k, v, n_heads: int, n_kv_heads: int) -> None:
    """Behind the model's own product: tensors as the model makes them, contiguous and of one device."""
    for t in (qkv, rope, positions, q, k, v):
        assert t.get_device() == qkv.get_device() and t.is_contiguous(), "contiguous tensors of one device"
    assert rows is None or (rows.get_device() == qkv.get_device() and rows.is_contiguous())
    call("mb8_rotate", qkv.get_device(), qkv.data_ptr(), rope.data_ptr(), positions.data_ptr(), None if rows is None else rows.data_ptr(), q.data_ptr(), k.data_ptr(), v.data_ptr(), qkv.shape[0],
         n_heads, n_kv_heads)
