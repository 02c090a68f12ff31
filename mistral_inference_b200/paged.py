"""Keys and values in pages of 8 bits: requests of different lengths share one pool instead of a rectangle of the longest one's length (cache.py), and each key costs
half of its 16-bit bytes to read.

  PageTables    which pages each request has: block tables, lengths and the free pages, on the GPU.  `extend` plans a step (block tables and slot map from the number
                of new tokens of each request), `truncate` takes tokens back.
  write_pages   keys and values of a plan's tokens into one layer's pool
  attend_pages  causal attention of a plan's tokens over that pool

A page holds 64 tokens of one request, for every key/value head: [2 (keys, values), 64, 128] e4m3 numbers and one power of two as scale for each head and kind.  All of
it runs in libmb200_paged.so (include/mistral_b200_paged.h)."""
from dataclasses import dataclass
from typing import Optional, Tuple

import torch

from . import _abi_paged
from ._abi import Mb200Error
from ._abi_paged import HEAD_DIM, PAGE

SOFTMAX_SCALE = HEAD_DIM ** -0.5
_REASONS = {1: "a row out of range, or named twice", 2: "a length that is negative or longer than a row of the block table", 3: "more tokens than the plan has room for",
            4: "too few free pages", 16: "a wait inside attention ran out", 32: "a request of more tokens than the plan's `most`"}


def pages_of(tokens: int) -> int:
    return -(-tokens // PAGE)


def check_status(status: torch.Tensor) -> None:
    """Raises if a plan's or a truncation's status says that it was refused (waits for the GPU)."""
    code = int(status)
    if code:
        raise Mb200Error("pages: " + "; ".join(v for k, v in _REASONS.items() if (code & k if k >= 16 else code & 15 == k)))


@dataclass
class PagePlan:
    """One step of B requests, for all layers (int32 tensors on the GPU)."""
    table: torch.Tensor      # [R, P] block table
    rows: torch.Tensor       # [B] each request's row of it
    q_start: torch.Tensor    # [B + 1] prefix sums of the new tokens
    seqpos: torch.Tensor     # [B] tokens that each request had before
    positions: torch.Tensor  # [T] position of each new token in its request
    slots: torch.Tensor      # [T] page * 64 + place in the page, -1: none
    longest: int             # no request has more new tokens
    most: int = 0            # no request has more tokens in all, the new ones among them (0: unknown)
    status: Optional[torch.Tensor] = None  # [1] 0, or why nothing was planned

    def check(self) -> "PagePlan":
        if self.status is not None:
            check_status(self.status)
        return self


class PageTables:
    """Block tables of up to R requests.  Tokens are planned and taken back on the current stream, without a copy from or to the host: calls can be captured in a graph."""

    def __init__(self, table: torch.Tensor, lens: torch.Tensor, free: torch.Tensor, n_free: torch.Tensor):
        """table [R, P] (page ids, -1 behind a row's last), lens [R], free [pages] of which the first n_free[0] are free (the last of them is taken first): int32, kept and
        written in place."""
        for t in (table, lens, free, n_free):
            assert t.dtype == torch.int32 and t.is_contiguous() and t.device == table.device, "contiguous int32 tensors of one device"
        assert table.dim() == 2 and lens.shape == table.shape[:1] and free.dim() == 1 and n_free.shape == (1,), (table.shape, lens.shape, free.shape, n_free.shape)
        self.table, self.lens, self.free, self.n_free = table, lens, free, n_free
        self.device = _abi_paged.index_of(table)
        self.scratch = torch.zeros(1 + table.shape[0], dtype=torch.int32, device=table.device)
        self._every = torch.arange(table.shape[0], dtype=torch.int32, device=table.device)
        self._first = {}  # number of requests -> their rows, where they are the first ones

    @staticmethod
    def empty(rows: int, max_pages: int, n_pages: int, device) -> "PageTables":
        """No tokens yet; pages are taken from 0 on."""
        i32 = dict(dtype=torch.int32, device=device)
        return PageTables(torch.full((rows, max_pages), -1, **i32), torch.zeros(rows, **i32), torch.arange(n_pages - 1, -1, -1, **i32), torch.full((1,), n_pages, **i32))

    def _requests(self, count: torch.Tensor, rows: Optional[torch.Tensor]) -> Tuple[torch.Tensor, torch.Tensor]:
        assert count.dtype is torch.int32 and count.dim() == 1 and count.shape[0] >= 1 and count.is_contiguous() and count.get_device() == self.device, f"one int32 a request, on cuda:{self.device}"
        if rows is None:
            B = count.shape[0]
            if B not in self._first:
                assert B <= self.table.shape[0], f"{B} requests, {self.table.shape[0]} rows"
                self._first[B] = self._every[:B]
            return count, self._first[B]
        assert rows.dtype is torch.int32 and rows.shape == count.shape and rows.is_contiguous() and rows.get_device() == self.device, "rows: one int32 a request"
        return count, rows

    def extend(self, add: torch.Tensor, n_tokens: int, rows: Optional[torch.Tensor] = None, longest: Optional[int] = None, most: int = 0) -> PagePlan:
        """Request b (row rows[b], or row b) takes add[b] more tokens, n_tokens in all at most; places of the plan behind the last new token stay empty (slot -1).  No
        request takes more than `longest`, none has more than `most` afterwards (both sizes of launches; unknown: n_tokens, a whole row).  A step that cannot be done changes nothing
        and leaves the reason in the plan's status: `plan.check()` raises it."""
        add, rows = self._requests(add, rows)
        B, T = add.shape[0], int(n_tokens)
        assert T >= 0
        block = torch.empty(2 * T + 2 * B + 2, dtype=torch.int32, device=self.table.device)
        positions, slots, q_start, seqpos, status = torch.split_with_sizes(block, (T, T, B + 1, B, 1))
        _abi_paged.pages_extend(self, rows, add, block, B, T)
        return PagePlan(self.table, rows, q_start, seqpos, positions, slots, max(1, T if longest is None else int(longest)), int(most), status)

    def truncate(self, keep: torch.Tensor, rows: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Request b keeps its first keep[b] tokens (0: it has ended).  Returns the status (see `check_status`)."""
        keep, rows = self._requests(keep, rows)
        status = torch.empty(1, dtype=torch.int32, device=self.table.device)
        _abi_paged.pages_truncate(self, rows, keep, status)
        return status


def empty_pool(n_pages: int, n_kv_heads: int, device) -> Tuple[torch.Tensor, torch.Tensor]:
    """(kv, scale) of one layer."""
    return (torch.zeros(n_pages, n_kv_heads, 2, PAGE, HEAD_DIM, dtype=torch.uint8, device=device).view(torch.float8_e4m3fn),
            torch.ones(n_pages, n_kv_heads, 2, dtype=torch.float32, device=device))


_I32, _CODES = torch.int32, (torch.float8_e4m3fn, torch.uint8)


def _pool(kv: torch.Tensor, scale: torch.Tensor, plan: PagePlan) -> Tuple[int, int, int]:
    """(device, pages, key/value heads) of a pool that a plan's tokens go into or attend over, all of it checked."""
    N, KV, kinds, tokens, dim = kv.shape
    dev = _abi_paged.index_of(kv)
    assert kinds == 2 and tokens == PAGE and dim == HEAD_DIM and kv.dtype in _CODES and kv.is_contiguous(), f"pool [pages, heads, 2, {PAGE}, {HEAD_DIM}] of e4m3, got {tuple(kv.shape)} {kv.dtype}"
    assert scale.shape == (N, KV, 2) and scale.dtype is torch.float32 and scale.is_contiguous() and scale.get_device() == dev, f"one fp32 scale for each page, head and kind, got {tuple(scale.shape)} {scale.dtype}"
    B = plan.rows.shape[0]
    assert plan.q_start.shape[0] == B + 1 and plan.seqpos.shape[0] == B and plan.longest >= 1, "a plan of PageTables.extend"
    for t in (plan.rows, plan.q_start, plan.seqpos, plan.slots):
        assert t.dtype is _I32 and t.get_device() == dev and t.is_contiguous(), f"plans are contiguous int32 tensors on cuda:{dev}, got {t.dtype} on {t.device}"
    return dev, N, KV


def write_pages(kv: torch.Tensor, scale: torch.Tensor, k: torch.Tensor, v: torch.Tensor, plan: PagePlan) -> None:
    """Keys and values [T, heads, 128] (or [T, heads * 128]; bf16) of the plan's tokens into the pool.  A page's scale for a head is the smallest power of two under which all
    of its tokens' numbers fit e4m3; it grows with later tokens.  Numbers that are not finite are kept as NaN."""
    dev, N, KV = _pool(kv, scale, plan)
    T = plan.slots.shape[0]
    assert k.shape[0] == T and v.shape[0] == T, f"{T} tokens planned, keys of {k.shape[0]}, values of {v.shape[0]}"
    if T:
        _abi_paged.pages_write(dev, kv, scale, k, v, plan, T, N, KV)


def attend_pages(q: torch.Tensor, kv: torch.Tensor, scale: torch.Tensor, plan: PagePlan, window: int = 0, softmax_scale: Optional[float] = None,
                 out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """[T, H * 128] bf16: attention of the queries [T, H, 128] (or [T, H * 128]; bf16) of the plan's tokens, whose own keys and values have been written before.  A query sees the
    last `window` positions of its request up to its own (0: all).  H is a multiple of the pool's heads, at most 32 times as many.  Rows of `out` behind the plan's last
    token stay as they are."""
    dev, N, KV = _pool(kv, scale, plan)
    T, width = q.shape[0], q.shape[1] * q.shape[2] if q.dim() == 3 else q.shape[1]
    assert T == plan.slots.shape[0], f"{plan.slots.shape[0]} tokens planned, queries {tuple(q.shape)}"
    H = width // HEAD_DIM
    assert width == H * HEAD_DIM and H >= 1 and H % KV == 0, f"{width} columns of queries, {KV} key/value heads"
    R, P = plan.table.shape
    assert plan.table.dtype is _I32 and plan.table.is_contiguous() and plan.table.get_device() == dev, f"block table: contiguous int32 on cuda:{dev}"
    if out is None:
        out = torch.empty((T, width), dtype=torch.bfloat16, device=kv.device)
    else:
        assert out.shape == (T, width) and out.dtype is torch.bfloat16 and out.is_contiguous() and out.get_device() == dev, f"out [T, {width}] bf16, got {tuple(out.shape)} {out.dtype}"
    if T:
        _abi_paged.attn_pages(dev, q, kv, scale, plan, out, T, N, KV, H, R, P, int(window), SOFTMAX_SCALE if softmax_scale is None else float(softmax_scale))
    return out
