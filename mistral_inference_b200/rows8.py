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
from ._abi_rows8 import BLOCK, MAX_NORM, MAX_ROWS

_E4M3, _E8M0, _BF16, _F32 = torch.float8_e4m3fn, torch.float8_e8m0fnu, torch.bfloat16, torch.float32


_empty = torch.empty_strided  # (half of the host's time of torch.empty with a shape)


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
        width, tiles = _width(cols), _tiles(rows, cols)
        return Rows8(_empty((rows, width), (width, 1), dtype=_E4M3, device=device), _empty(tiles, (tiles[1] * 512, 512, 16, 4, 1), dtype=_E8M0, device=device), cols)

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
        return (self.codes.float().view(self.rows, -1, BLOCK) * power[:, :, None]).view(self.rows, -1)[:, : self.cols].to(dtype)


def _check_rows8(x: Rows8, what: str) -> Tuple[int, int]:
    """(device, rows) of a matrix in this form, all of it checked."""
    c, s, cols = x.codes, x.scales, x.cols
    shape = c.shape
    assert len(shape) == 2 and c.dtype is _E4M3 and s.dtype is _E8M0 and cols >= 1 and shape[1] == _width(cols) and s.shape == _tiles(shape[0], cols), \
        f"{what}: codes [rows, {_width(cols)}] e4m3 and scales {_tiles(len(c), cols)} e8m0, got {tuple(shape)} {c.dtype} and {tuple(s.shape)} {s.dtype}"
    dev = c.get_device()
    assert dev >= 0, f"libmb200_rows8 runs on CUDA only (got {c.device}); no fallback exists"
    assert s.get_device() == dev and c.is_contiguous() and s.is_contiguous(), f"{what}: contiguous codes and scales of one device"
    return dev, shape[0]


def _check_numbers(x: torch.Tensor, what: str) -> Tuple[int, int, int, int]:
    """(device, rows, columns, elements from row to row)"""
    shape, dtype = x.shape, x.dtype
    assert len(shape) == 2 and (dtype is _BF16 or dtype is _F32) and shape[1] >= 1, f"{what} [rows, columns], bf16 or fp32, got {tuple(shape)} {dtype}"
    T, K = shape
    ld, step = x.stride()
    assert (step == 1 or K == 1) and (ld >= K or T <= 1), f"{what}: contiguous rows that do not overlap"
    dev = x.get_device()
    assert dev >= 0, f"libmb200_rows8 runs on CUDA only (got {x.device}); no fallback exists"
    return dev, T, K, ld


def quantise_rows(x: torch.Tensor) -> Rows8:
    """Rows of x [T, K] (bf16 or fp32; rows may be part of wider ones) as 8-bit numbers.  The power of a block of 128 is 2^e, e >= -100 the smallest with max |x| <= 448 * 2^e; numbers
    are rounded to nearest, ties to even.  A block that holds a NaN or an infinity becomes NaN."""
    dev, T, K, ld = _check_numbers(x, "x")
    out = Rows8.empty(T, K, x.device)
    _abi_rows8.call("mb8_quantise", dev, x.data_ptr(), ld, 1 if x.dtype is _F32 else 0, out.codes.data_ptr(), out.scales.data_ptr(), T, K)
    return out


def norm_rows(x: torch.Tensor, weight: torch.Tensor, eps: float, add: Optional[torch.Tensor] = None) -> Tuple[Rows8, torch.Tensor]:
    """(rows, h): h = x + add in x's type (x itself without `add`), rows = h * rsqrt(mean(h^2) + eps) * weight as 8-bit numbers (the statistics and the products are fp32; no rounding to 16
    bits in between).  x, add [T, K] (rows may be part of wider ones), weight [K], all bf16 or all fp32."""
    dev, T, K, ld = _check_numbers(x, "x")
    dtype = x.dtype
    assert K <= MAX_NORM, f"rows of {K} entries (at most {MAX_NORM})"
    assert weight.dtype is dtype and weight.shape == (K,) and weight.is_contiguous() and weight.get_device() == dev, f"weight [{K}] {dtype} on {x.device}"
    out = Rows8.empty(T, K, x.device)
    wide = 1 if dtype is _F32 else 0
    if add is None:
        _abi_rows8.call("mb8_norm", dev, x.data_ptr(), ld, None, 0, weight.data_ptr(), wide, None, out.codes.data_ptr(), out.scales.data_ptr(), T, K, eps)
        return out, x
    add_dev, add_T, add_K, ld_add = _check_numbers(add, "add")
    assert add.dtype is dtype and add_T == T and add_K == K and add_dev == dev, f"add {(T, K)} {dtype} on {x.device}"
    h = _empty((T, K), (K, 1), dtype=dtype, device=x.device)
    _abi_rows8.call("mb8_norm", dev, x.data_ptr(), ld, add.data_ptr(), ld_add, weight.data_ptr(), wide, h.data_ptr(), out.codes.data_ptr(), out.scales.data_ptr(), T, K, eps)
    return out, h


def multiply_rows(x: Rows8, w: Rows8, dtype: torch.dtype = torch.bfloat16, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """x [T, K] times w [N, K] transposed: [T, N] bf16 or fp32, summed in fp32 and rounded once.  `out`: results of the caller's, rows may be part of wider ones."""
    dev, T = _check_rows8(x, "x")
    w_dev, N = _check_rows8(w, "w")
    assert w_dev == dev and x.cols == w.cols and N >= 1, f"rows of one length on one device, got {x.cols} and {N} of {w.cols}"
    if out is None:
        assert dtype is _BF16 or dtype is _F32, f"bf16 or fp32 results, got {dtype}"
        out, ld = _empty((T, N), (N, 1), dtype=dtype, device=x.codes.device), N
    else:
        out_dev, out_T, out_N, ld = _check_numbers(out, "out")
        assert out_T == T and out_N == N and out_dev == dev, f"out [{T}, {N}] on {x.codes.device}"
        dtype = out.dtype
    _abi_rows8.product("mb8_multiply", dev, x, w, (out.data_ptr(), ld, 1 if dtype is _F32 else 0), T, N, N)
    return out


def gate_rows(x: Rows8, w13: Rows8) -> Rows8:
    """silu(x w1^T) * (x w3^T) of x [T, K] as 8-bit numbers [T, H]: row 2 i of w13 [2 H, K] is w1's row i, row 2 i + 1 is w3's."""
    dev, T = _check_rows8(x, "x")
    w_dev, N = _check_rows8(w13, "w13")
    assert w_dev == dev and x.cols == w13.cols and N >= 2 and N % 2 == 0, f"pairs of rows of one length on one device, got {x.cols} and {N} of {w13.cols}"
    out = Rows8.empty(T, N // 2, x.codes.device)
    _abi_rows8.product("mb8_gate", dev, x, w13, (out.codes.data_ptr(), out.scales.data_ptr()), T, N, N // 2)
    return out
