"""Plain 64-bit restatements of the paged operators and of token scores, on the CPU, page by page and query by query."""
import math
from typing import List, Optional

import torch

PAGE, HD = 64, 128
E4M3 = torch.float8_e4m3fn


def cdiv(a: int, b: int) -> int:
    return -(-a // b)


class HostTables:
    """The state of block tables in Python lists."""

    def __init__(self, rows: int, max_pages: int, n_pages: int):
        self.table = [[-1] * max_pages for _ in range(rows)]
        self.lens = [0] * rows
        self.free = list(range(n_pages - 1, -1, -1))  # the whole array; the first n_free are free
        self.n_free = n_pages

    def extend(self, add: List[int], rows: Optional[List[int]] = None):
        rows = list(range(len(add))) if rows is None else rows
        positions, slots, q_start, seqpos = [], [], [0], []
        for r, n in zip(rows, add):
            seqpos.append(self.lens[r])
            for j in range(cdiv(self.lens[r], PAGE), cdiv(self.lens[r] + n, PAGE)):
                self.n_free -= 1
                self.table[r][j] = self.free[self.n_free]
            for pos in range(self.lens[r], self.lens[r] + n):
                positions.append(pos)
                slots.append(self.table[r][pos // PAGE] * PAGE + pos % PAGE)
            self.lens[r] += n
            q_start.append(q_start[-1] + n)
        return positions, slots, q_start, seqpos

    def truncate(self, keep: List[int], rows: Optional[List[int]] = None) -> None:
        rows = list(range(len(keep))) if rows is None else rows
        back = []
        for r, n in zip(rows, keep):
            for j in range(cdiv(n, PAGE), cdiv(self.lens[r], PAGE)):
                back.append(self.table[r][j])
                self.table[r][j] = -1
            self.lens[r] = n
        for page in reversed(back):
            self.free[self.n_free] = page
            self.n_free += 1


def e4m3_grid() -> torch.Tensor:
    """All finite e4m3 numbers from 0 up, in 64 bits: by exponent and mantissa."""
    out = [m * 2.0 ** -9 for m in range(8)]
    for e in range(-6, 9):
        out += [(8 + m) * 2.0 ** (e - 3) for m in range(8)]
    return torch.tensor(out[:-1], dtype=torch.float64)  # the last pattern is NaN


def to_e4m3(x: torch.Tensor) -> torch.Tensor:
    """The nearest e4m3 number (64 bits, |x| <= 448), the even code where two are as near; NaN for what is not finite."""
    grid = e4m3_grid()
    a = x.abs().nan_to_num(0.0, 0.0, 0.0)
    hi = torch.searchsorted(grid, a).clamp(max=len(grid) - 1)
    lo = (hi - 1).clamp(min=0)
    below, above = a - grid[lo], grid[hi] - a
    code = torch.where((above < below) | ((above == below) & (hi % 2 == 0)), hi, lo)
    return torch.where(x.isfinite(), torch.copysign(grid[code], x), math.nan)


def page_exponent(amax: float) -> int:
    e = -100
    while amax > 448.0 * 2.0 ** e:
        e += 1
    return e


def write_ref(kv: torch.Tensor, scale: torch.Tensor, k: torch.Tensor, v: torch.Tensor, slots: List[int]) -> None:
    """kv [pages, KV, 2, 64, 128] and scale in 64 bits, in place; k, v [T, KV, 128]."""
    x = torch.stack([k, v], 2).double()
    t = 0
    while t < len(slots):
        if slots[t] < 0:
            t += 1
            continue
        page, off = divmod(slots[t], PAGE)
        n = 1
        while t + n < len(slots) and slots[t + n] == slots[t] + n and off + n < PAGE:
            n += 1
        for g in range(kv.shape[1]):
            for kind in range(2):
                new = x[t:t + n, g, kind]
                fine = new[new.isfinite()].abs()
                e = page_exponent(float(fine.max()) if fine.numel() else 0.0)
                if off:
                    old = round(math.log2(float(scale[page, g, kind])))
                    e = max(e, old)
                    if e > old:
                        kv[page, g, kind, :off] = to_e4m3(kv[page, g, kind, :off] * 2.0 ** (old - e))
                scale[page, g, kind] = 2.0 ** e
                kv[page, g, kind, off:off + n] = to_e4m3(new / 2.0 ** e)
        t += n


def attend_ref(q: torch.Tensor, kv: torch.Tensor, scale: torch.Tensor, table, rows, q_start, seqpos, window: int = 0, softmax_scale: Optional[float] = None):
    """(o [T, H, 128], A [T, H, 128]) in 64 bits: the attention, and the same weights over the values' magnitudes.  q [T, H, 128]; only what a query sees is read."""
    T, H, _ = q.shape
    KV = kv.shape[1]
    out, mag = torch.zeros(T, H, HD, dtype=torch.float64), torch.zeros(T, H, HD, dtype=torch.float64)
    f = HD ** -0.5 if softmax_scale is None else softmax_scale
    for b, r in enumerate(rows):
        for i in range(q_start[b + 1] - q_start[b]):
            pos, t = seqpos[b] + i, q_start[b] + i
            first = max(0, pos - window + 1) if window else 0
            at = torch.arange(first, pos + 1)
            page = torch.tensor([table[r][j] for j in range(cdiv(pos + 1, PAGE))])[at // PAGE]
            x = kv.double()[page, :, :, at % PAGE] * scale.double()[page][..., None]  # [keys, KV, 2, 128]
            k, v = (x[:, :, kind].repeat_interleave(H // KV, 1) for kind in range(2))
            s = torch.einsum("hd,khd->hk", q[t].double(), k) * f
            w = torch.softmax(s, 1)
            out[t] = torch.einsum("hk,khd->hd", w, v)
            mag[t] = torch.einsum("hk,khd->hd", w, v.abs())
    return out, mag


def attend_tolerance(want: torch.Tensor, mag: torch.Tensor, keys: int, vmax: float) -> torch.Tensor:
    """How far the kernel may be.  The result is rounded to bf16 once: 2^-8 of it.  Each weight is given to the tensor cores as hi + lo / 16 in e4m3: hi is off by at most 2^-4 of
    the weight, lo by 2^-4 of that, 2^-8 in all, of the weights' share of the values' magnitudes; a weight so small that its parts are subnormal is off by at most 2^-10 / 16 of
    e4m3's units, where the largest is 256: 2^-22 of the largest weight, each of `keys`.  Scores are fp32 sums of exact products (a query's two parts hold its 8 bits; below 2^-14 of a
    row's largest entry they are off by at most 2^-23 of that): for |q k| sums up to 2^6 in units of the exponent, 2 * 128 * 2^-24 * 2^6 = 2^-10 at the very worst relative to a weight,
    numerator and denominator both."""
    return 2.0 ** -8 * want.abs() + (2.0 ** -8 + 2.0 ** -9) * mag * (1 + 2.0 ** -8) + keys * 2.0 ** -22 * vmax


def scores_ref(logits: torch.Tensor, targets, top: int):
    """(logprob [T], entropy [T], ids [T, top], logprobs [T, top]) in 64 bits; ranked by a stable sort."""
    lp_out, ent, ids, lps = [], [], [], []
    for t, row in enumerate(logits.double().cpu()):
        bad = bool(row.isnan().any()) or bool((row == math.inf).any()) or bool((row == -math.inf).all())
        # the largest entry's 1 stays out of the sum: 64 bits beside it would keep only 2^-53 / S of a small rest S
        rest = row.clone()
        rest[row.nan_to_num(-math.inf).argmax()] = -math.inf
        m = row.max()
        lp = row - m - torch.log1p(torch.exp(rest - m).sum())
        rank = torch.where(row.isnan(), math.inf, row)  # (rows of NaN hold no infinity in these tests)
        order = torch.sort(rank + 0.0, descending=True, stable=True).indices[:top]
        p = lp.exp()
        nan = torch.tensor(math.nan, dtype=torch.float64)
        ent.append(nan if bad else -(p * lp)[p > 0].sum())
        ids.append(order)
        lps.append(torch.full((top,), math.nan, dtype=torch.float64) if bad else lp[order])
        if targets is not None:
            i = int(targets[t])
            lp_out.append(torch.zeros((), dtype=torch.float64) if i < 0 else nan if bad or i >= row.numel() else lp[i])
    return torch.stack(lp_out) if targets is not None else None, torch.stack(ent), torch.stack(ids), torch.stack(lps)
