"""Linears of 8-bit numbers: half of the weight bytes that a decode step reads, and twice the tensor cores' rate for prompts.

  Rows8          a matrix whose rows are e4m3 codes with a power of two for every 128 of them: weights [out, in] and activations [tokens, in] alike
  quantise_rows  16- or 32-bit rows in that form
  norm_rows      the root-mean-square norm of a residual stream in that form, with the addition to the stream ahead of it
  multiply_rows  x W^T to 16 or 32 bits
  gate_rows      silu(x W1^T) * (x W3^T) in that form again, the two weights' rows interleaved

All of it runs in libmb200_rows8.so (include/mistral_b200_rows8.h).  `Transformer.quantise_weights()` keeps a model's Linears in this form."""
from dataclasses import dataclass
from typing import Optional, Tuple

import torch

from . import _abi_rows8
from ._abi_rows8 import BLOCK, MAX_ROWS

_E4M3, _E8M0, _BF16, _F32 = torch.float8_e4m3fn, torch.float8_e8m0fnu, torch.bfloat16, torch.float32


def _width(cols: int) -> int:
    return -(-cols // BLOCK) * BLOCK


def _tiles(rows: int, cols: int) -> Tuple[int, int, int, int, int]:
    return (rows + 127) // 128, (cols + 4 * BLOCK - 1) // (4 * BLOCK), 32, 4, 4


@dataclass(eq=False)
class Rows8:
    """[rows, cols] numbers: code * power."""
    codes: torch.Tensor   # [rows, cols rounded up to 128] float8_e4m3fn, zeros behind a row's end
    scales: torch.Tensor  # [ceil(rows / 128), ceil(cols / 512), 32, 4, 4] float8_e8m0fnu: row 32 j + i and block c of a tile at [i, j, c]; 1 where there is no row or block
    cols: int
    fixed: bool = False   # everything that ever wrote it has ended (a loaded model's weights): products may read it before their turn on their stream

    @property
    def rows(self) -> int:
        return self.codes.shape[0]

    @staticmethod
    def empty(rows: int, cols: int, device) -> "Rows8":
        """Not yet written."""
        assert 0 <= rows <= MAX_ROWS and 1 <= cols <= MAX_ROWS, f"{rows} rows of {cols} entries (at most {MAX_ROWS})"
        return Rows8(torch.empty(rows, _width(cols), dtype=_E4M3, device=device), torch.empty(_tiles(rows, cols), dtype=_E8M0, device=device), cols)

    def to(self, device) -> "Rows8":
        """On another device (itself where it is there already)."""
        codes = self.codes.to(device)
        return self if codes is self.codes else Rows8(codes, self.scales.to(device), self.cols)

    def _blocks(self, tiles: torch.Tensor) -> torch.Tensor:
        """Bytes in tiles as [rows, blocks]."""
        n, quads = tiles.shape[:2]
        return tiles.permute(0, 3, 2, 1, 4).reshape(n * 128, quads * 4)[: self.rows, : self.codes.shape[1] // BLOCK]

    def exponents(self) -> torch.Tensor:
        """[rows, ceil(cols / 128)] int32: the power of two of each block."""
        return self._blocks(self.scales.view(torch.uint8)).int() - 127

    def numbers(self, dtype: torch.dtype = torch.float32) -> torch.Tensor:
        """[rows, cols]: what the codes stand for (exact in 16 bits as well)."""
        power = self._blocks(self.scales.view(torch.uint8)).contiguous().view(_E8M0).float()
        return (self.codes.float().view(self.rows, power.shape[1], BLOCK) * power[:, :, None]).view(self.codes.shape)[:, : self.cols].to(dtype)


_host = None  # the extension that checks, allocates and launches (csrc/rows8/rows8_host.cpp), once a call needed it


def _load():
    global _host
    _host = _abi_rows8.host()
    return _host


def quantise_rows(x: torch.Tensor) -> Rows8:
    """Rows of x [T, K] (bf16 or fp32; rows may be part of wider ones) as 8-bit numbers.  The power of a block of 128 is 2^e, e >= -100 the smallest with max |x| <= 448 * 2^e; numbers
    are rounded to nearest, ties to even.  A block that holds a NaN or an infinity becomes NaN."""
    codes, scales = (_host or _load()).quantise(x)
    return Rows8(codes, scales, x.shape[1])


def norm_rows(x: torch.Tensor, weight: torch.Tensor, eps: float, add: Optional[torch.Tensor] = None) -> Tuple[Rows8, torch.Tensor]:
    """(rows, h): h = x + add in x's type (x itself without `add`), rows = h * rsqrt(mean(h^2) + eps) * weight as 8-bit numbers (the statistics and the products are fp32; no rounding to 16
    bits in between).  x, add [T, K] (rows may be part of wider ones, at most 65536 columns), weight [K], all bf16 or all fp32."""
    codes, scales, h = (_host or _load()).norm(x, weight, eps, add)
    return Rows8(codes, scales, x.shape[1]), x if h is None else h


def multiply_rows(x: Rows8, w: Rows8, dtype: Optional[torch.dtype] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """x [T, K] times w [N, K] transposed: [T, N] bf16 (without `dtype`) or fp32, summed in fp32 and rounded once.  `out`: results of the caller's, of its type; rows may be part of wider ones."""
    assert dtype is None or dtype is _BF16 or dtype is _F32, f"bf16 or fp32 results, got {dtype}"
    assert out is None or dtype is None or getattr(out, "dtype", dtype) is dtype, f"results of type {dtype}, and out of another"
    return (_host or _load()).multiply(x.codes, x.scales, x.cols, w.codes, w.scales, w.cols, w.fixed, dtype is _F32, out)


def gate_rows(x: Rows8, w13: Rows8) -> Rows8:
    """silu(x w1^T) * (x w3^T) of x [T, K] as 8-bit numbers [T, H]: row 2 i of w13 [2 H, K] is w1's row i, row 2 i + 1 is w3's."""
    codes, scales = (_host or _load()).gate(x.codes, x.scales, x.cols, w13.codes, w13.scales, w13.cols, w13.fixed)
    return Rows8(codes, scales, w13.codes.shape[0] // 2)
