"""The 4-bit cache and the attention over it by their definitions, in 64 bits and number by number: what the tests of the
kernels and of the engine compare with.  Nothing here uses the package."""

import math

import torch

MAGNITUDE = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)


def scale_of(byte: int) -> float:
    if byte == 255:
        return math.nan
    e, m = byte >> 3, byte & 7
    return m * 2.0 ** -17 if e == 0 else (8 + m) * 2.0 ** (e - 18)


SCALES = torch.tensor([scale_of(b) for b in range(256)], dtype=torch.float64)


def quantized(x: torch.Tensor) -> torch.Tensor:
    """What the cache holds for ``x`` ``[..., D]``, float64: the nearest scale of all scales, the nearest number of all numbers."""
    g = x.double().unflatten(-1, (-1, 16))
    top = g.abs().amax(-1)
    usable = SCALES[:227]
    want = (top / 6.0).clamp(max=10240.0)
    # nearest of the 227 scales, ties to the even byte
    above = torch.searchsorted(usable, want.contiguous()).clamp(max=226)
    below = (above - 1).clamp(min=0)
    up, down = usable[above] - want, want - usable[below]
    byte = torch.where((up < down) | ((up == down) & (above % 2 == 0)), above, below)
    scale = torch.where(top.isfinite(), usable[byte], torch.full_like(want, math.nan))[..., None]
    ratio = torch.where(scale > 0, g.abs() / scale, torch.zeros_like(g)).clamp(max=8.0)
    off = (ratio[..., None] - MAGNITUDE).abs()
    near = off.amin(-1, keepdim=True)
    odd_last = torch.where(off == near, torch.arange(8) % 2, 2)                # of two at the same distance the even code
    code = odd_last.argmin(-1)
    return (torch.where(g < 0, -1.0, 1.0) * MAGNITUDE[code] * scale).flatten(-2)


def decoded(pages: torch.Tensor, D: int) -> torch.Tensor:
    """Pages ``[pages, KV, records, 9 D]`` -> float64 ``[pages, KV, records * 16, D]``."""
    raw = pages.cpu()
    codes = raw[..., :8 * D].unflatten(-1, (16, D // 2)).long()
    nibble = torch.stack([codes % 16, codes // 16], -1).flatten(-2)
    scale = SCALES[raw[..., 8 * D:].unflatten(-1, (16, D // 16)).long()].repeat_interleave(16, -1)
    return (torch.where(nibble >= 8, -1.0, 1.0) * MAGNITUDE[nibble % 8] * scale).flatten(2, 3)


def attention(q, k_pages, v_pages, table, q_start, kv_len, page, scale, window):
    """float64 ``[T, H, D]``, and the largest magnitude of a score and of a value met."""
    T, H, D = q.shape
    k_all, v_all = decoded(k_pages, D), decoded(v_pages, D)
    KV = k_all.shape[1]
    out = torch.zeros((T, H, D), dtype=torch.float64)
    most_s = most_v = 0.0
    q, table, q_start, kv_len = q.double().cpu(), table.cpu(), q_start.tolist(), kv_len.tolist()
    for b, L in enumerate(kv_len):
        n = q_start[b + 1] - q_start[b]
        for i in range(n):
            pos = L - n + i
            if pos < 0:
                continue
            keys = torch.arange(max(0, pos - window + 1) if window else 0, pos + 1)
            pages = table[b][keys // page].long()
            assert (pages >= 0).all()
            for h in range(H):
                k, v = k_all[pages, h // (H // KV), keys % page], v_all[pages, h // (H // KV), keys % page]
                s = k @ q[q_start[b] + i, h] * scale
                out[q_start[b] + i, h] = torch.softmax(s, 0) @ v
                most_s, most_v = max(most_s, float(s.abs().max())), max(most_v, float(v.abs().max()))
    return out, most_s, most_v
