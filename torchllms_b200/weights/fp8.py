"""Rows of numbers in 8 bits: the value type, and the format in plain PyTorch.

A row of ``K`` numbers (``K`` a multiple of 16) is ``K`` numbers of E4M3 and a scale, a power of two, for every 128 neighbouring ones.
With ``a`` the largest finite magnitude of the 128 the scale is ``2^e``, ``e`` the least integer with ``a <= 448 * 2^e``, at least -126
and at most 120 (-126 where ``a`` is 0); a number is divided by it, which is exact, and rounded to nearest, ties to even.  What is
not finite is held as NaN.  So the one rounding is E4M3's: half a unit of four significant bits, 2^-4 relative, down to
2^-6 * 2^e, and 2^-10 * 2^e absolute below.

A weight ``[N, K]`` of a product is ``N`` such rows, as the activations that it meets are; the weights of ``E`` experts are
``[E, N, K]``.  A scale of a power of two costs nothing in accuracy, since the numbers under it are floating, and it is what the
tensor cores' block-scaled instruction multiplies by, so sums stay where they are from block to block.

The reference has no weights below 16 bits (torchllms/models/networks.py:474-493, :592-605); this format is an addition.
``csrc/fp8.cuh`` has the kernels' side.  The functions below are for loading weights, for tools and for tests.
"""

from __future__ import annotations

import math
from dataclasses import dataclass
from typing import Tuple

import torch

BLOCK = 128                  # numbers that share a scale
WORD = 4                     # a row's scales come in whole words: 4 scales, 512 numbers
ALIGN = 16                   # a row is a multiple of so many numbers
MAX_NORM_WIDTH = 32768       # numbers of a row behind a norm (it stays in registers)
WEIGHT_FORMATS = ("full", "fp8")

CODES, SCALES = torch.float8_e4m3fn, torch.float8_e8m0fnu


def scale_pitch(width: int) -> int:
    """Scales that a row of ``width`` numbers has, the places behind the last (byte 0) among them."""
    return WORD * -(-width // (WORD * BLOCK))


def check_width(width: int, what: str = "8-bit rows") -> None:
    if width <= 0 or width % ALIGN != 0:
        raise ValueError(f"{what} take a multiple of {ALIGN} numbers a row, got {width}")


@dataclass(slots=True)
class Fp8Rows:
    """``codes`` ``[..., rows, K]`` (float8_e4m3fn) and ``scales`` ``[..., rows, scale_pitch(K)]`` (float8_e8m0fnu)."""

    codes: torch.Tensor
    scales: torch.Tensor

    @property
    def shape(self) -> torch.Size:
        return self.codes.shape

    @property
    def device(self) -> torch.device:
        return self.codes.device

    def __getitem__(self, rows: slice) -> "Fp8Rows":
        """Some of the rows (or of the experts): a view."""
        return Fp8Rows(self.codes[rows], self.scales[rows])

    def nbytes(self) -> int:
        return self.codes.numel() + self.scales.numel()

    def dequantize(self, dtype: torch.dtype = torch.float32) -> torch.Tensor:
        """What the rows stand for (exact in float32, and in bfloat16 as far as its range goes)."""
        return decode(self.codes, self.scales).to(dtype)


def encode(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """``[..., K]`` -> codes ``[..., K]`` and scales ``[..., scale_pitch(K)]``."""
    check_width(x.shape[-1])
    g = torch.nn.functional.pad(x.float(), (0, -x.shape[-1] % BLOCK)).unflatten(-1, (-1, BLOCK))
    fine = torch.isfinite(g)
    top = torch.where(fine, g.abs(), torch.zeros_like(g)).amax(-1)
    part, power = torch.frexp(top)                                  # top = part 2^power, part in [0.5, 1)
    e = torch.where(part <= 0.875, power - 9, power - 8).clamp(-126, 120)
    byte = (torch.where(top == 0, torch.full_like(e, -126), e) + 127).to(torch.uint8)
    scale = byte.view(SCALES).float()[..., None]
    codes = torch.where(fine, g / scale, torch.full_like(g, math.nan)).to(CODES)
    pad = scale_pitch(x.shape[-1]) - byte.shape[-1]
    return codes.flatten(-2)[..., :x.shape[-1]].contiguous(), torch.nn.functional.pad(byte, (0, pad)).view(SCALES)


def decode(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """What codes and scales stand for, float32."""
    width = codes.shape[-1]
    scale = scales.float()[..., :-(-width // BLOCK)].repeat_interleave(BLOCK, -1)[..., :width]
    return codes.float() * scale
