"""The 4-bit format of cached keys and values: sizes, and the numbers in plain PyTorch.

Sixteen neighbouring coordinates of a token's key (or value) of one head share a byte of scale and are held as a sign and one
of 0, 0.5, 1, 1.5, 2, 3, 4, 6 each (E2M1).  The scale has 5 bits of exponent and 3 of mantissa and no sign:
``M 2^-17`` for exponent 0, else ``(8 + M) 2^(E - 18)``.  With ``a`` the group's largest magnitude it is ``a / 6`` rounded to
nearest (ties to even), at most 10240; a number is divided by it and rounded to nearest (ties to the even code), at most 6.  So
numbers up to 61440 are held, and a group whose numbers are all below 6 * 2^-18 reads as zeros.  A group with a number that
is not finite gets scale byte 255 and reads as NaN.

Sixteen tokens of a head are a *record* of ``9 * head_dim`` bytes: 16 rows of ``head_dim / 2`` bytes (coordinate ``2 i`` in the
low half of byte ``i``), then 16 rows of ``head_dim / 16`` scales.  Page tensors are
``[pages, kv_heads, page_size / 16, 9 * head_dim]`` uint8.

The reference keeps keys and values in the model's dtype (torchllms/models/paged_kv.py:186-222); this format is an addition:
4.5 bits a number, so that the memory of a bfloat16 cache holds 3.6 times the tokens, and a decode step reads as much less.
``csrc/fp4.cuh`` has the kernels' side.  The functions below are for tools and tests; the engine does not call them.
"""

from __future__ import annotations

from typing import Tuple

import torch

CACHE_FORMATS = ("full", "fp4")
GROUP = 16           # coordinates that share a scale
RECORD = 16          # tokens of a record
TOP_SCALE = 226      # the scale byte of 10240, the largest
NAN_SCALE = 255
MAX_HEAD_DIM = 256   # what the attention kernels take


def check_head_dim(head_dim: int) -> None:
    if head_dim % GROUP != 0 or not GROUP <= head_dim <= MAX_HEAD_DIM:
        raise ValueError(f"a 4-bit cache takes heads of a multiple of {GROUP} coordinates up to {MAX_HEAD_DIM}, got {head_dim}")


def check_page_size(page_size: int) -> None:
    if page_size < RECORD or page_size % RECORD != 0:
        raise ValueError(f"a 4-bit cache takes pages of a multiple of {RECORD} tokens, got {page_size}")


def record_bytes(head_dim: int) -> int:
    return RECORD * (head_dim // 2 + head_dim // GROUP)


def page_shape(n_pages: int, n_kv_heads: int, page_size: int, head_dim: int) -> Tuple[int, int, int, int]:
    check_head_dim(head_dim)
    check_page_size(page_size)
    return (n_pages, n_kv_heads, page_size // RECORD, record_bytes(head_dim))


def encode(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """``[..., head_dim]`` -> bytes of numbers ``[..., head_dim / 2]`` and of scales ``[..., head_dim / 16]``."""
    g = x.float().unflatten(-1, (-1, GROUP))
    top = g.abs().amax(-1)
    want = top / torch.full((), 6.0, device=x.device)           # (by a tensor: a true division, not a product with 1/6)
    mantissa, exponent = torch.frexp(want)                       # want = mantissa 2^exponent, mantissa in [0.5, 1)
    normal = (mantissa * 16.0).round().int() + ((exponent + 13) << 3)      # 8 .. 16 eighths: the 16 carries into the exponent
    byte = torch.where(want < 2.0 ** -14, (want * 2.0 ** 17).round().int(), normal).clamp(0, TOP_SCALE)
    byte = torch.where(top.isfinite(), byte, torch.full_like(byte, NAN_SCALE))
    scale = scale_values(x.device)[byte.long()]
    usable = (byte > 0) & (byte != NAN_SCALE)
    a = torch.where(usable[..., None], g / torch.where(usable, scale, torch.ones_like(scale))[..., None], torch.zeros_like(g))
    m = a.abs()
    # nearest of the eight magnitudes, ties to the even code
    code = torch.where(m < 2.0, (2.0 * m).round(), torch.where(m < 4.0, m.round() + 2.0, (m / 2.0).round() + 4.0)).clamp(max=7.0).int()
    code = code + 8 * torch.signbit(a).int()
    pair = code.flatten(-2).unflatten(-1, (-1, 2))
    return (pair[..., 0] | (pair[..., 1] << 4)).to(torch.uint8), byte.to(torch.uint8)


def decode(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """What these bytes stand for, float32 ``[..., head_dim]``."""
    magnitude = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=codes.device)
    numbers = torch.cat([magnitude, -magnitude])
    nibbles = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).long()
    return numbers[nibbles] * scale_values(codes.device)[scales.long()].repeat_interleave(GROUP, -1)


def scale_values(device) -> torch.Tensor:
    """The scale of every byte."""
    byte = torch.arange(256, device=device)
    exponent, mantissa = byte >> 3, (byte & 7).float()
    scale = torch.where(exponent == 0, mantissa * 2.0 ** -17, (8.0 + mantissa) * torch.exp2((exponent - 18).float()))
    scale[NAN_SCALE] = float("nan")
    return scale


def rows_of(pages: torch.Tensor, head_dim: int) -> Tuple[torch.Tensor, torch.Tensor]:
    """Views of a page tensor: numbers ``[pages, kv_heads, page_size / 16, 16, head_dim / 2]`` and scales ``[.., 16, head_dim / 16]``."""
    at = RECORD * head_dim // 2
    return (pages[..., :at].unflatten(-1, (RECORD, head_dim // 2)), pages[..., at:].unflatten(-1, (RECORD, head_dim // GROUP)))


def store(pages: torch.Tensor, x: torch.Tensor, slots: torch.Tensor, page_size: int) -> None:
    """``x`` ``[n, kv_heads, head_dim]`` into the slots (``page * page_size + offset``) of a page tensor."""
    slots = slots.long()
    for view, value in zip(rows_of(pages, x.shape[-1]), encode(x)):
        view[slots // page_size, :, slots % page_size // RECORD, slots % RECORD] = value


def load(pages: torch.Tensor, slots: torch.Tensor, page_size: int, head_dim: int) -> torch.Tensor:
    """The numbers of these slots, float32 ``[n, kv_heads, head_dim]``."""
    slots = slots.long()
    return decode(*(view[slots // page_size, :, slots % page_size // RECORD, slots % RECORD] for view in rows_of(pages, head_dim)))
