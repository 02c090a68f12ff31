"""Rows of 8-bit numbers restated in 64 bits, element by element of the definition."""
import math

import torch

BLOCK, MAX, LOWEST = 128, 448.0, -100


def power(e: torch.Tensor) -> torch.Tensor:
    """2^e in 64 bits, exactly."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def blocks_of(x: torch.Tensor) -> torch.Tensor:
    """[T, K] as [T, blocks, 128] in 64 bits, zeros behind the end."""
    T, K = x.shape
    out = torch.zeros(T, -(-K // BLOCK) * BLOCK, dtype=torch.float64, device=x.device)
    out[:, :K] = x.double()
    return out.view(T, -1, BLOCK)


def exponent(amax: torch.Tensor) -> torch.Tensor:
    """The smallest e >= LOWEST with amax <= 448 * 2^e; 0 where amax is no number (the block is NaN)."""
    powers = torch.tensor([MAX * 2.0 ** e for e in range(LOWEST, 128)], dtype=torch.float64, device=amax.device)
    e = torch.searchsorted(powers, amax.contiguous()) + LOWEST
    return torch.where(amax.isfinite(), e, torch.zeros_like(e))


def tiles_of(e: torch.Tensor) -> torch.Tensor:
    """Bytes of exponents [T, blocks] in their tiles."""
    T, n = e.shape
    out = torch.full((-(-T // 128), -(-n // 4), 32, 4, 4), 127, dtype=torch.uint8, device=e.device)
    for r in range(0, T, 32):
        for b in range(n):
            rows = e[r:r + 32, b]
            out[r // 128, b // 4, : rows.shape[0], r % 128 // 32, b % 4] = (rows + 127).to(torch.uint8)
    return out


def quantised(x: torch.Tensor):
    """(codes [T, width] e4m3, bytes of scales in tiles) of rows of numbers."""
    b = blocks_of(x)
    nan = ~b.isfinite().all(2)
    e = exponent(torch.where(nan[:, :, None], torch.zeros_like(b), b).abs().amax(2))
    e = torch.where(nan, torch.zeros_like(e), e)
    scaled = b * power(-e)[:, :, None]
    scaled = torch.where(nan[:, :, None], torch.full_like(scaled, math.nan), scaled)
    # (the conversion takes 32-bit numbers: these have at most 24 bits and are within their range)
    return scaled.float().to(torch.float8_e4m3fn).view(x.shape[0], -1), tiles_of(e)


def numbers(codes: torch.Tensor, scales: torch.Tensor, cols: int) -> torch.Tensor:
    """What codes and scales in tiles stand for, in 64 bits."""
    T, width = codes.shape
    bytes_ = scales.view(torch.uint8)
    r, b = torch.meshgrid(torch.arange(T, device=codes.device), torch.arange(width // BLOCK, device=codes.device), indexing="ij")
    size = power(bytes_[r // 128, b // 4, r % 32, r % 128 // 32, b % 4].long() - 127)
    return (codes.double().view(T, -1, BLOCK) * size[:, :, None]).view(T, width)[:, :cols]


def product(x: torch.Tensor, w: torch.Tensor):
    """(y, bound) of x [T, K] times w [N, K] transposed, of numbers in 64 bits.  The products of two e4m3 numbers are exact in 32 bits.  32 of them are added at a time to a 32-bit sum;
    each of these additions is taken to be off by at most 2^-21 of the magnitudes that it adds (numbers aligned to the largest, and some bits cut off)."""
    y, size = x @ w.t(), x.abs() @ w.abs().t()
    return y, size * (-(-x.shape[1] // 32) * 2.0 ** -21)


def assert_rows_near(codes, scales, y, off, what=""):
    """Codes and scales are those of rows y [T, K] that may be off by `off` before they are rounded: powers exactly those of numbers within that distance, and every number within half a
    step (2^-4 of it, or 2^-10 of the power among the smallest) behind it."""
    T, K = y.shape
    off = torch.as_tensor(off, dtype=torch.float64, device=y.device).expand(T, K)
    b, o = blocks_of(y), blocks_of(off)
    least, most = exponent((b.abs() - o).clamp(min=0).amax(2)), exponent((b.abs() + o).amax(2))
    bytes_ = scales.view(torch.uint8)
    n = b.shape[1]
    r, c = torch.meshgrid(torch.arange(T, device=y.device), torch.arange(n, device=y.device), indexing="ij")
    e = bytes_[r // 128, c // 4, r % 32, r % 128 // 32, c % 4].long() - 127
    assert ((e >= least) & (e <= most)).all(), what
    expect = tiles_of(e)
    assert torch.equal(bytes_, expect), f"{what}: places of no row or block hold 127"
    got = codes.double() * power(e).repeat_interleave(BLOCK, 1)
    assert (got[:, K:] == 0).all(), what
    step = torch.maximum((y.abs() + off) * 2.0 ** -4, power(e - 10).repeat_interleave(BLOCK, 1)[:, :K])
    bad = (got[:, :K] - y).abs() > off + step
    assert not bad.any(), f"{what}: {int(bad.sum())} numbers off, the first at {bad.nonzero()[0].tolist()}"
