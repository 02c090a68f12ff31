"""ctypes binding of libmb200_paged.so (C ABI: include/mistral_b200_paged.h): pages of 8-bit keys and values, scores of tokens.

Same rules as `_abi`: the only place Python touches this library, and no fallback -- a missing library is built once
in-tree by `build.build_paged()` (a fresh checkout has no binaries), a failing call raises.
"""
import contextlib
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
    "mbp_attn_pages_scratch": (I, [I, I, I, I, I, I, I]),
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


def _ptr(t: Optional[torch.Tensor], device: torch.device) -> Optional[int]:
    if t is None:
        return None
    assert t.device == device and t.is_contiguous(), f"libmb200_paged takes contiguous tensors of one device ({device}, got one on {t.device})"
    return t.data_ptr()


def _on(device: torch.device):
    """The library works on the current device: make it the tensors' own."""
    assert device.type == "cuda", f"libmb200_paged runs on CUDA only (got {device}); no fallback exists"
    return contextlib.nullcontext() if device.index == torch.cuda.current_device() else torch.cuda.device(device)


def _rows(x: torch.Tensor, heads: int, device: torch.device) -> Tuple[int, int]:
    """(pointer, elements between tokens) of [T, heads, 128] or [T, heads * 128] bf16; tokens may be rows of a wider matrix."""
    assert x.dtype == torch.bfloat16 and x.device == device, f"bf16 tokens on {device}, got {x.dtype} on {x.device}"
    if x.dim() == 3:
        assert x.shape[1:] == (heads, HEAD_DIM) and x.stride(2) == 1 and (heads == 1 or x.stride(1) == HEAD_DIM), f"[T, {heads}, {HEAD_DIM}] with contiguous heads, got {tuple(x.shape)}"
    else:
        assert x.dim() == 2 and x.shape[1] == heads * HEAD_DIM and x.stride(1) == 1, f"[T, {heads * HEAD_DIM}] with contiguous rows, got {tuple(x.shape)}"
    width = heads * HEAD_DIM
    return x.data_ptr(), x.stride(0) if x.shape[0] > 1 else width


def pages_extend(tables, rows, add, positions, slots, q_start, seqpos, status, T: int) -> None:
    dev = tables.table.device
    R, width = tables.table.shape
    with _on(dev):
        _check(lib().mbp_pages_extend(_ptr(tables.table, dev), _ptr(tables.lens, dev), _ptr(tables.free, dev), _ptr(tables.n_free, dev), _ptr(tables.scratch, dev), _ptr(rows, dev),
                                      _ptr(add, dev), _ptr(positions, dev), _ptr(slots, dev), _ptr(q_start, dev), _ptr(seqpos, dev), _ptr(status, dev), add.shape[0], T, R, width,
                                      tables.free.shape[0], _stream()), "mbp_pages_extend")


def pages_truncate(tables, rows, keep, status) -> None:
    dev = tables.table.device
    R, width = tables.table.shape
    with _on(dev):
        _check(lib().mbp_pages_truncate(_ptr(tables.table, dev), _ptr(tables.lens, dev), _ptr(tables.free, dev), _ptr(tables.n_free, dev), _ptr(tables.scratch, dev), _ptr(rows, dev),
                                        _ptr(keep, dev), _ptr(status, dev), keep.shape[0], R, width, tables.free.shape[0], _stream()), "mbp_pages_truncate")


def pages_write(kv, scale, k, v, plan) -> None:
    dev, KV = kv.device, kv.shape[1]
    pk, ldk = _rows(k, KV, dev)
    pv, ldv = _rows(v, KV, dev)
    with _on(dev):
        _check(lib().mbp_pages_write(pk, ldk, pv, ldv, _ptr(kv, dev), _ptr(scale, dev), _ptr(plan.slots, dev), _ptr(plan.q_start, dev), _ptr(plan.seqpos, dev), plan.rows.shape[0],
                                     plan.slots.shape[0], KV, HEAD_DIM, kv.shape[0], _stream()), "mbp_pages_write")


@functools.lru_cache(maxsize=256)
def _attn_scratch(B: int, longest: int, most: int, width: int, n_heads: int, KV: int, window: int) -> int:
    return lib().mbp_attn_pages_scratch(B, longest, most, width, n_heads, KV, window)


def attn_pages(q, kv, scale, plan, out, n_heads: int, window: int, softmax_scale: float) -> None:
    dev, KV = kv.device, kv.shape[1]
    pq, ldq = _rows(q, n_heads, dev)
    R, width = plan.table.shape
    B = plan.rows.shape[0]
    need = _attn_scratch(B, plan.longest, plan.most, width, n_heads, KV, window)
    with _on(dev):
        scratch = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
        _check(lib().mbp_attn_pages(pq, ldq, _ptr(kv, dev), _ptr(scale, dev), _ptr(plan.table, dev), _ptr(plan.rows, dev), _ptr(plan.q_start, dev), _ptr(plan.seqpos, dev), _ptr(out, dev),
                                    _ptr(plan.status, dev), B, q.shape[0], plan.longest, plan.most, R, width, kv.shape[0], n_heads, KV, HEAD_DIM, window, softmax_scale,
                                    None if scratch is None else scratch.data_ptr(), need, _stream()), "mbp_attn_pages")


@functools.lru_cache(maxsize=256)
def _scores_scratch(T: int, V: int, top: int) -> int:
    need = c_int64(0)
    _check(lib().mbp_token_scores_sizes(T, V, top, ctypes.byref(need)), "mbp_token_scores_sizes")
    return need.value


def token_scores(logits, targets, logprob, entropy, top_ids, top_logprobs, top: int) -> None:
    T, V = logits.shape
    dev = logits.device
    with _on(dev):
        scratch = torch.empty(_scores_scratch(T, V, top), dtype=torch.uint8, device=dev)
        _check(lib().mbp_token_scores(logits.data_ptr(), logits.stride(0) if T > 1 else V, 1 if logits.dtype == torch.float32 else 0, _ptr(targets, dev), _ptr(logprob, dev), _ptr(entropy, dev),
                                      _ptr(top_ids, dev), _ptr(top_logprobs, dev), T, V, top, scratch.data_ptr(), _stream()), "mbp_token_scores")
