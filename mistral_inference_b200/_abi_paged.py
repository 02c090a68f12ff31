"""ctypes binding of libmb200_paged.so (C ABI: include/mistral_b200_paged.h): pages of 8-bit keys and values, scores of tokens.

Same rules as `_abi`: the only place Python touches this library, and no fallback -- a missing library is built once
in-tree by `build.build_paged()` (a fresh checkout has no binaries), a failing call raises.
"""
import ctypes
import functools
from ctypes import c_char_p, c_float, c_int, c_int64, c_void_p
from typing import Optional, Tuple

import torch

from . import build
from ._abi import Mb200Error, _stream

ABI_VERSION = 1
PAGE = 64       # tokens of a page
HEAD_DIM = 128
MAX_REQUESTS = 4000
MAX_TOP = 64
MAX_SCORE_ROWS = 65535  # rows of a call
_lib: Optional[ctypes.CDLL] = None

P, I = c_void_p, c_int64
_SIGNATURES = {
    "mbp_abi_version": (c_int, []),
    "mbp_last_error": (c_char_p, []),
    "mbp_pages_extend": (c_int, [P, P, P, P, P, P, P, P, P, P, P, P, I, I, I, I, I, P]),
    "mbp_pages_truncate": (c_int, [P, P, P, P, P, P, P, P, I, I, I, I, P]),
    "mbp_pages_write": (c_int, [P, I, P, I, P, P, P, P, P, I, I, I, I, I, P]),
    "mbp_attn_pages_scratch": (I, [I, I, I, I, I, I, I, I]),
    "mbp_attn_pages": (c_int, [P, I, P, P, P, P, P, P, P, P, I, I, I, I, I, I, I, I, I, I, I, c_float, P, I, P]),
    "mbp_token_scores_sizes": (c_int, [I, I, I, P]),
    "mbp_token_scores": (c_int, [P, I, c_int, P, P, P, P, P, I, I, I, P, P]),
}


def lib() -> ctypes.CDLL:
    global _lib
    if _lib is None:
        handle = ctypes.CDLL(str(build.build_paged()))
        for name, (restype, argtypes) in _SIGNATURES.items():
            fn = getattr(handle, name)
            fn.restype, fn.argtypes = restype, argtypes
        if handle.mbp_abi_version() != ABI_VERSION:
            raise Mb200Error(f"libmb200_paged ABI {handle.mbp_abi_version()} != expected {ABI_VERSION}")
        _lib = handle
    return _lib


def _check(rc: int, what: str) -> None:
    if rc != 0:
        msg = lib().mbp_last_error()
        raise Mb200Error(f"{what} failed ({rc}): {msg.decode() if msg else '?'}")


_lazy = {}  # name -> entry point, once the library is loaded


def _fn(name: str):
    fn = _lazy.get(name)
    if fn is None:
        fn = _lazy[name] = getattr(lib(), name)
    return fn


def index_of(t: torch.Tensor) -> int:
    """The device that a call works on: its tensors' own, whatever the current one is."""
    i = t.get_device()
    assert i >= 0, f"libmb200_paged runs on CUDA only (got {t.device}); no fallback exists"
    return i


def _ptr(t: Optional[torch.Tensor], device: int) -> Optional[int]:
    if t is None:
        return None
    assert t.get_device() == device and t.is_contiguous(), f"libmb200_paged takes contiguous tensors of one device (cuda:{device}, got one on {t.device})"
    return t.data_ptr()


def _call(name: str, device: int, *args) -> None:
    """The entry point on the current stream of `device`, whatever the current device is."""
    fn = _fn(name)
    if device == torch._C._cuda_getDevice():
        rc = fn(*args, _stream())
    else:
        with torch.cuda.device(device):
            rc = fn(*args, _stream())
    if rc != 0:
        _check(rc, name)


def _rows(x: torch.Tensor, heads: int, device: int) -> Tuple[int, int]:
    """(pointer, elements between tokens) of [T, heads, 128] or [T, heads * 128] bf16; tokens may be rows of a wider matrix."""
    assert x.dtype == torch.bfloat16 and x.get_device() == device, f"bf16 tokens on cuda:{device}, got {x.dtype} on {x.device}"
    shape, stride = x.shape, x.stride()
    if len(shape) == 3:
        assert shape[1] == heads and shape[2] == HEAD_DIM and stride[2] == 1 and (heads == 1 or stride[1] == HEAD_DIM), f"[T, {heads}, {HEAD_DIM}] with contiguous heads, got {tuple(shape)}"
    else:
        assert len(shape) == 2 and shape[1] == heads * HEAD_DIM and stride[1] == 1, f"[T, {heads * HEAD_DIM}] with contiguous rows, got {tuple(shape)}"
    return x.data_ptr(), stride[0] if shape[0] > 1 else heads * HEAD_DIM


def _state(tables):
    return tables.table.data_ptr(), tables.lens.data_ptr(), tables.free.data_ptr(), tables.n_free.data_ptr(), tables.scratch.data_ptr()


def pages_extend(tables, rows, add, block, B: int, T: int) -> None:
    """block: positions [T] | slots [T] | q_start [B + 1] | seqpos [B] | status [1]."""
    at = block.data_ptr()
    R, width = tables.table.shape
    _call("mbp_pages_extend", tables.device, *_state(tables), rows.data_ptr(), add.data_ptr(), at, at + 4 * T, at + 8 * T, at + 8 * T + 4 * (B + 1), at + 8 * T + 4 * (2 * B + 1), B, T, R,
          width, tables.free.shape[0])


def pages_truncate(tables, rows, keep, status) -> None:
    R, width = tables.table.shape
    _call("mbp_pages_truncate", tables.device, *_state(tables), rows.data_ptr(), keep.data_ptr(), status.data_ptr(), keep.shape[0], R, width, tables.free.shape[0])


def pages_write(dev: int, kv, scale, k, v, plan, T: int, N: int, KV: int) -> None:
    pk, ldk = _rows(k, KV, dev)
    pv, ldv = _rows(v, KV, dev)
    _call("mbp_pages_write", dev, pk, ldk, pv, ldv, kv.data_ptr(), scale.data_ptr(), plan.slots.data_ptr(), plan.q_start.data_ptr(), plan.seqpos.data_ptr(), plan.rows.shape[0], T, KV,
          HEAD_DIM, N)


@functools.lru_cache(maxsize=256)
def _attn_scratch(device: int, B: int, T: int, longest: int, most: int, width: int, n_heads: int, KV: int, window: int) -> int:
    """How a call is cut goes by its device's SMs: the same device is asked that the call will run on."""
    with torch.cuda.device(device):
        return _fn("mbp_attn_pages_scratch")(B, T, longest, most, width, n_heads, KV, window)


def attn_pages(dev: int, q, kv, scale, plan, out, T: int, N: int, KV: int, H: int, R: int, width: int, window: int, softmax_scale: float) -> None:
    pq, ldq = _rows(q, H, dev)
    B, status = plan.rows.shape[0], plan.status
    need = _attn_scratch(dev, B, T, plan.longest, plan.most, width, H, KV, window)
    scratch = torch.empty(need, dtype=torch.uint8, device=kv.device) if need else None
    _call("mbp_attn_pages", dev, pq, ldq, kv.data_ptr(), scale.data_ptr(), plan.table.data_ptr(), plan.rows.data_ptr(), plan.q_start.data_ptr(), plan.seqpos.data_ptr(), out.data_ptr(),
          None if status is None else _ptr(status, dev), B, T, plan.longest, plan.most, R, width, N, H, KV, HEAD_DIM, window, softmax_scale, None if scratch is None else scratch.data_ptr(), need)


@functools.lru_cache(maxsize=256)
def _scores_scratch(T: int, V: int, top: int) -> int:
    need = c_int64(0)
    _check(lib().mbp_token_scores_sizes(T, V, top, ctypes.byref(need)), "mbp_token_scores_sizes")
    return need.value


def token_scores(logits, targets, logprob, entropy, top_ids, top_logprobs, top: int) -> None:
    T, V = logits.shape
    dev = index_of(logits)
    scratch = logits.new_empty(_scores_scratch(T, V, top) // 4 + 2, dtype=torch.float32)  # (of 8 bytes' alignment, as any)
    _call("mbp_token_scores", dev, logits.data_ptr(), logits.stride(0) if T > 1 else V, 1 if logits.dtype == torch.float32 else 0, _ptr(targets, dev), _ptr(logprob, dev), _ptr(entropy, dev),
          _ptr(top_ids, dev), _ptr(top_logprobs, dev), T, V, top, scratch.data_ptr())
