"""Keys and values in pages of 8 bits: requests of different lengths share one pool instead of a rectangle of the longest one's length (cache.py), and each key costs
half of its 16-bit bytes to read.

  PageTables    which pages each request has: block tables, lengths and the free pages, on the GPU.  `extend` plans a step (block tables and slot map from the number
                of new tokens of each request), `truncate` takes tokens back.
  write_pages   keys and values of a plan's tokens into one layer's pool
  attend_pages  causal attention of a plan's tokens over that pool
  PagedCache    pools of all layers with their block tables, in the place of a BufferCache: `Transformer.make_cache(..., kv_cache="pages")`

A page holds 64 tokens of one request, for every key/value head: [2 (keys, values), 64, 128] e4m3 numbers and one power of two as scale for each head and kind.  All of
it runs in libmb200_paged.so (include/mistral_b200_paged.h)."""
from dataclasses import dataclass
from typing import List, Optional, Tuple

import torch

from . import _abi_paged
from ._abi import Mb200Error
from ._abi_paged import HEAD_DIM, PAGE
from .cache import SlidingWindow, get_cache_sizes, upload

SOFTMAX_SCALE = HEAD_DIM ** -0.5
_REASONS = {1: "a row out of range, or named twice", 2: "a length that is negative or longer than a row of the block table", 3: "more tokens than the plan has room for",
            4: "too few free pages, or a number of them that the stack cannot have", 16: "a wait inside attention ran out", 32: "a request of more tokens than the plan's `longest` or `most`"}


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
        self.scratch = torch.zeros(1, dtype=torch.int32, device=table.device)
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
        block = self.lens.new_empty(2 * T + 2 * B + 2)
        positions, slots, q_start, seqpos, status = torch.unsafe_split_with_sizes(block, (T, T, B + 1, B, 1))
        _abi_paged.pages_extend(self, rows, add, block, B, T)
        return PagePlan(self.table, rows, q_start, seqpos, positions, slots, max(1, T if longest is None else int(longest)), int(most), status)

    def truncate(self, keep: torch.Tensor, rows: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Request b keeps its first keep[b] tokens (0: it has ended).  Returns the status (see `check_status`)."""
        keep, rows = self._requests(keep, rows)
        status = self.lens.new_empty(1)
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
    of its tokens' numbers fit e4m3; it grows with later tokens (and keeps that if they are taken back).  Numbers that are not finite are kept as NaN.  Plans are written in the
    order in which they were made."""
    dev, N, KV = _pool(kv, scale, plan)
    T = plan.slots.shape[0]
    assert k.shape[0] == T and v.shape[0] == T, f"{T} tokens planned, keys of {k.shape[0]}, values of {v.shape[0]}"
    if T:
        _abi_paged.pages_write(dev, kv, scale, k, v, plan, T, N, KV)


def attend_pages(q: torch.Tensor, kv: torch.Tensor, scale: torch.Tensor, plan: PagePlan, window: int = 0, softmax_scale: Optional[float] = None,
                 out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """[T, H * 128] bf16: attention of the queries [T, H, 128] (or [T, H * 128]; bf16) of the plan's tokens, whose own keys and values have been written before.  A query sees the
    last `window` positions of its request up to its own (0: all).  H is a multiple of the pool's heads, at most 32 times as many.  Rows of `out` behind the plan's last
    token stay as they are.  A NaN among the values makes its column NaN for the queries that see it; in a portion long enough to go through 16-bit rings also for
    others of its block of 128 tokens, as in the prompt kernel."""
    dev, N, KV = _pool(kv, scale, plan)
    T, width = q.shape[0], q.shape[1] * q.shape[2] if q.dim() == 3 else q.shape[1]
    assert T == plan.slots.shape[0], f"{plan.slots.shape[0]} tokens planned, queries {tuple(q.shape)}"
    H = width // HEAD_DIM
    assert width == H * HEAD_DIM and H >= 1 and H % KV == 0, f"{width} columns of queries, {KV} key/value heads"
    R, P = plan.table.shape
    assert plan.table.dtype is _I32 and plan.table.is_contiguous() and plan.table.get_device() == dev, f"block table: contiguous int32 on cuda:{dev}"
    if out is None:
        out = q.new_empty(T, width)
    else:
        assert out.shape == (T, width) and out.dtype is torch.bfloat16 and out.is_contiguous() and out.get_device() == dev, f"out [T, {width}] bf16, got {tuple(out.shape)} {out.dtype}"
    if T:
        _abi_paged.attn_pages(dev, q, kv, scale, plan, out, T, N, KV, H, R, P, int(window), SOFTMAX_SCALE if softmax_scale is None else float(softmax_scale))
    return out


class PageLedger:
    """The host's account of a PagedCache: which row each live request has, its tokens, and how many pages are free.  It knows before a step is launched whether there is room."""

    def __init__(self, rows: int, max_seq_len: int, n_pages: int):
        self.max_seq_len, self.n_pages = max_seq_len, n_pages
        self.free_rows = list(range(rows - 1, -1, -1))
        self.rows: List[int] = []  # of the live requests, in batch order
        self.lens: List[int] = []  # their tokens

    @property
    def free_pages(self) -> int:
        return self.n_pages - sum(pages_of(n) for n in self.lens)

    def admit(self, n: int) -> None:
        if n > len(self.free_rows):
            raise ValueError(f"{n} more requests in a cache with {len(self.free_rows)} free rows")
        for _ in range(n):
            self.rows.append(self.free_rows.pop())
            self.lens.append(0)

    def retire(self, indices: List[int]) -> None:
        gone = set(indices)
        assert all(0 <= i < len(self.rows) for i in gone), indices
        self.free_rows += [self.rows[i] for i in sorted(gone, reverse=True)]
        keep = [i for i in range(len(self.rows)) if i not in gone]
        self.rows, self.lens = [self.rows[i] for i in keep], [self.lens[i] for i in keep]

    def check(self, seqlens: List[int]) -> None:
        """Raises if the live requests cannot take so many more tokens each."""
        if len(seqlens) != len(self.rows):
            raise ValueError(f"Batch size is {len(self.rows)}, got {len(seqlens)}, did you forget to reset cache?")
        if min(seqlens) < 0 or sum(seqlens) < 1:
            raise ValueError(f"new tokens of each request: {seqlens}")
        if max(n + a for n, a in zip(self.lens, seqlens)) > self.max_seq_len:
            raise ValueError(f"a request of more than {self.max_seq_len} tokens")
        need = sum(pages_of(n + a) - pages_of(n) for n, a in zip(self.lens, seqlens))
        if need > self.free_pages:
            raise ValueError(f"{need} more pages needed, {self.free_pages} of {self.n_pages} free")


@dataclass
class PagedInputMetadata:
    """What one layer's kernels need for this forward (CacheInputMetadata's part for pages)."""
    plan: PagePlan
    positions: torch.Tensor
    q_start: torch.Tensor
    seqpos: torch.Tensor
    prefill: bool
    first_prefill: bool  # nothing cached before for any request
    seqlens: List[int]
    max_seqlen: int
    window: int          # positions that a query sees, itself included


class PagedView:
    """One layer's pool plus the metadata of this forward."""
    paged = True

    def __init__(self, kv: torch.Tensor, scale: torch.Tensor, metadata: PagedInputMetadata, windowed: bool):
        self.kv, self.scale, self.metadata, self.windowed = kv, scale, metadata, windowed

    def write(self, k: torch.Tensor, v: torch.Tensor) -> None:
        write_pages(self.kv, self.scale, k, v, self.metadata.plan)

    def attend(self, q: torch.Tensor, out: torch.Tensor) -> torch.Tensor:
        return attend_pages(q, self.kv, self.scale, self.metadata.plan, window=self.metadata.window if self.windowed else 0, out=out)


class PagedCache:
    """Keys and values of a running batch in 8-bit pages, with a BufferCache's methods for `Transformer.forward` and `generate()`.  Requests take pages as they grow and share
    n_pages of them (by default as many as all rows of max_seq_len tokens need); they can be retired from a running batch and others admitted to it (`seqlens` of a
    forward then has a 0 for those that bring nothing).  A request's pages are kept for its whole length, also behind a sliding window."""
    paged = True

    def __init__(self, n_layers: int, max_batch_size: int, max_seq_len: int, n_kv_heads: int, head_dim: int, sliding_window: SlidingWindow = None, n_pages: Optional[int] = None,
                 device: torch.device = torch.device("cuda")):
        assert head_dim == HEAD_DIM, f"pages hold heads of {HEAD_DIM} dimensions, got {head_dim}"
        assert max_batch_size <= _abi_paged.MAX_REQUESTS, f"at most {_abi_paged.MAX_REQUESTS} requests"
        self.n_layers, self.max_batch_size, self.max_seq_len, self.n_kv_heads, self.head_dim = n_layers, max_batch_size, max_seq_len, n_kv_heads, head_dim
        self.cache_sizes = get_cache_sizes(n_layers, max_seq_len, sliding_window)
        self.windowed = [w is not None for w in (sliding_window * (n_layers // len(sliding_window)) if isinstance(sliding_window, list) else [sliding_window] * n_layers)]
        each = pages_of(max_seq_len)
        self.n_pages = max_batch_size * each if n_pages is None else n_pages
        self.tables = PageTables.empty(max_batch_size, each, self.n_pages, device)
        self.pools = [empty_pool(self.n_pages, n_kv_heads, device) for _ in range(n_layers)]
        self.reset()

    # -- the batch ------------------------------------------------------------------------------
    def reset(self) -> None:
        """No requests: every page is free."""
        t = self.tables
        t.table.fill_(-1)
        t.lens.zero_()
        t.free.copy_(torch.arange(self.n_pages - 1, -1, -1, dtype=torch.int32))
        t.n_free.fill_(self.n_pages)
        self.ledger = PageLedger(self.max_batch_size, self.max_seq_len, self.n_pages)
        self._on_device: List[int] = []  # tokens of the live requests in the block tables (a forward that failed may have left more than the ledger says)
        self._rows_dev: Optional[torch.Tensor] = None
        self._started = False
        self.__dict__.pop("_mb200_decode_states", None)

    def init_kvseqlens(self, batch_size: int) -> None:
        assert not self._started, "a batch is running: reset() first, or admit() more requests"
        self.admit(batch_size)

    def _batch_changed(self) -> None:
        self._rows_dev = None
        self.__dict__.pop("_mb200_decode_states", None)  # captured decode graphs are per batch size and row set

    def admit(self, n: int = 1) -> List[int]:
        """n more requests, without tokens yet; their places in the batch order (the last ones)."""
        self.ledger.admit(n)
        self._on_device += [0] * n
        self._started = True
        self._batch_changed()
        return list(range(len(self.ledger.rows) - n, len(self.ledger.rows)))

    def retire(self, indices: List[int]) -> None:
        """Requests `indices` (places in the batch order) have ended: their pages and rows are free, the others keep their order."""
        gone = sorted(set(indices))
        rows = [self.ledger.rows[i] for i in gone]
        self.ledger.retire(gone)
        if rows:
            self.tables.truncate(self._ints([0] * len(rows)), self._ints(rows))
        self._on_device = [n for i, n in enumerate(self._on_device) if i not in set(gone)]
        self._batch_changed()

    @property
    def rows(self) -> List[int]:
        return self.ledger.rows

    @property
    def _kv_seqlens_host(self) -> Optional[List[int]]:
        return self.ledger.lens if self._started else None

    @property
    def kv_seqlens(self) -> Optional[torch.Tensor]:
        return torch.tensor(self.ledger.lens, device=self.device, dtype=torch.long) if self._started else None

    @property
    def device(self) -> torch.device:
        return self.tables.table.device

    def update_seqlens(self, seqlens: List[int]) -> None:
        """After a forward: its tokens count.  Negative numbers take (drafted) tokens back."""
        assert len(seqlens) == len(self.ledger.lens), f"{len(seqlens)} numbers of tokens, {len(self.ledger.lens)} requests"
        lens = [n + a for n, a in zip(self.ledger.lens, seqlens)]
        assert all(0 <= n <= d for n, d in zip(lens, self._on_device)), (self.ledger.lens, seqlens)
        self.ledger.lens = lens

    # -- metadata ---------------------------------------------------------------------------------
    def _ints(self, values: List[int]) -> torch.Tensor:
        return upload(torch.tensor(values, dtype=torch.int32), self.device)

    def rows_on_device(self) -> torch.Tensor:
        if self._rows_dev is None:
            self._rows_dev = self._ints(self.ledger.rows)
        return self._rows_dev

    def settle(self) -> None:
        """Tokens that the ledger does not count leave the block tables."""
        if self._on_device != self.ledger.lens:
            self.tables.truncate(self._ints(self.ledger.lens), self.rows_on_device())
            self._on_device = list(self.ledger.lens)

    def planned(self, seqlens: List[int]) -> None:
        """The block tables hold `seqlens` more tokens of each request, or are about to (planned here, or by a step that is run or replayed next): settle() takes back what a
        failed step has left of them, and finds nothing to take back where it never came to its plan."""
        self._on_device = [n + a for n, a in zip(self.ledger.lens, seqlens)]

    def metadata_of(self, plan: PagePlan, seqlens: List[int], first: bool) -> List[PagedInputMetadata]:
        """One per layer (shared by layers of one window).  first: no request has a token yet, and attention need not read pages; a step that is captured may be replayed when
        they have some."""
        longest = max(seqlens)
        per_w = {w: PagedInputMetadata(plan, plan.positions, plan.q_start, plan.seqpos, first or longest > 1, first, list(seqlens), longest, w) for w in set(self.cache_sizes)}
        return [per_w[w] for w in self.cache_sizes]

    def get_input_metadata(self, seqlens: List[int]) -> List[PagedInputMetadata]:
        seqlens = [int(n) for n in seqlens]
        if not self._started:
            self.init_kvseqlens(len(seqlens))
        self.ledger.check(seqlens)
        self.settle()
        most = max(n + a for n, a in zip(self.ledger.lens, seqlens))
        plan = self.tables.extend(self._ints(seqlens), sum(seqlens), self.rows_on_device(), longest=max(seqlens), most=most)
        self.planned(seqlens)
        return self.metadata_of(plan, seqlens, first=not any(self.ledger.lens))

    def get_view(self, layer_id: int, metadata: PagedInputMetadata) -> PagedView:
        kv, scale = self.pools[layer_id]
        return PagedView(kv, scale, metadata, self.windowed[layer_id])
