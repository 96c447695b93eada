"""The 8-bit rows and what is done with them, from the definitions, in 64 bits: what the kernels are held to."""

import math

import torch

BLOCK = 128


def pitch(width):
    return 4 * -(-width // 512)


def hold(x):
    """64-bit ``[rows, K]`` -> the numbers that are held (before their scale) and the exponents ``[rows, ceil(K / 128)]``."""
    R, K = x.shape
    g = torch.zeros((R, -(-K // BLOCK) * BLOCK), dtype=torch.float64, device=x.device)
    g[:, :K] = x.double()
    g = g.reshape(R, g.shape[1] // BLOCK, BLOCK)
    fine = torch.isfinite(g)
    a = torch.where(fine, g.abs(), torch.zeros_like(g)).amax(-1, keepdim=True)
    e = torch.ceil(torch.log2((a / 448.0).clamp(min=2.0 ** -126)))
    e = torch.where(a > 448.0 * torch.exp2(e), e + 1, torch.where((a <= 448.0 * torch.exp2(e - 1)) & (e > -126), e - 1, e))
    v = torch.where(fine, g, torch.zeros_like(g)) / torch.exp2(e)
    quantum = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6))) - 3)
    held = torch.where(fine, (v / quantum).round() * quantum, torch.full_like(g, math.nan))
    return held.flatten(1)[:, :K], e[..., 0]


def value(rows):
    """What an ``Fp8Rows`` stands for, 64 bits."""
    K = rows.codes.shape[-1]
    return rows.codes.double() * rows.scales.double().repeat_interleave(BLOCK, -1)[..., :K]


def stands_for(x):
    held, e = hold(x)
    return held * torch.exp2(e).repeat_interleave(BLOCK, -1)[:, :x.shape[1]]


def act(u, kind, gated=False, params=None):
    """Activations of the feed-forwards in 64 bits."""
    if gated:
        g, up = u.chunk(2, -1)
        if kind == "clamped_swish":
            limit, alpha, offset = params
            g, up = g.clamp(max=limit), up.clamp(-limit, limit)
            return g * torch.sigmoid(alpha * g) * (up + offset)
        return act(g, kind) * up
    if kind == "silu":
        return u * torch.sigmoid(u)
    if kind == "gelu_tanh":
        return 0.5 * u * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (u + 0.044715 * u ** 3)))
    if kind == "gelu":
        return 0.5 * u * (1.0 + torch.erf(u / math.sqrt(2.0)))
    assert kind == "relu2"
    return u.clamp(min=0) ** 2


def experts(x, chosen, weights, up, down, kind, gated=False, params=None):
    """``sum_k weights * down(act(up x))`` with the rows held in 8 bits on the way, 64 bits; ``up`` and ``down`` 64-bit ``[E, ..]``."""
    rows = stands_for(x.double())
    out = torch.zeros_like(rows)
    for e in range(up.shape[0]):
        token, choice = torch.nonzero(chosen == e, as_tuple=True)
        if token.numel():
            y = stands_for(act(rows[token] @ up[e].T, kind, gated, params)) @ down[e].T
            out.index_add_(0, token, y * weights[token, choice].double()[:, None])
    return out


def moved(y, d):
    """How far what ``y`` is held as may move when ``y`` moves by ``d`` (both 64-bit ``[rows, K]``): a number next to a border of E4M3 falls to
    its other side, and where a block's largest number stands next to the border of its scale, the small ones get another step."""
    at = stands_for(y)
    reach = torch.maximum((stands_for(y + d) - at).abs(), (stands_for(y - d) - at).abs())
    e = torch.exp2(hold(y)[1])
    pad = lambda v: torch.nn.functional.pad(v, (0, -v.shape[1] % BLOCK)).reshape(v.shape[0], -1, BLOCK).amax(-1)  # noqa: E731
    top, slack = pad(y.abs()), pad(d)
    border = (top + slack > 448.0 * e) | ((top - slack) <= 224.0 * e)
    return reach + (border * e * 2.0 ** -8).repeat_interleave(BLOCK, -1)[:, :y.shape[1]]


def activated(x, w, kind, gated=False, params=None):
    """``act(x @ w.T)`` and how far float32 arithmetic may be from it: the sums are off by 2^-24 of their magnitudes for every 32 terms (and 4
    more), the activation by what that does to it, at the corners, and by 2^-20 of itself and 2^-21 of its argument's size."""
    u = x @ w.T
    du = (x.abs() @ w.abs().T) * (x.shape[1] / 32 + 4) * 2.0 ** -24
    y = act(u, kind, gated, params)
    if gated:
        half = u.shape[1] // 2
        sides = [torch.cat([a * du[:, :half], b * du[:, half:]], 1) for a in (-1, 1) for b in (-1, 1)]
        size = u[:, :half].abs() * (u[:, half:].abs() + 1.0)
    else:
        sides, size = [-du, du], u.abs()
    return y, torch.stack([(act(u + s, kind, gated, params) - y).abs() for s in sides]).amax(0) + y.abs() * 2.0 ** -20 + size * 2.0 ** -21


def experts_bound(x, chosen, weights, up, down, kind, gated=False, params=None, result_eps=0.0):
    """How far a result of float32 arithmetic may be from :func:`experts`, for every number of it: the hidden numbers as in :func:`activated`;
    each is then held as it is, or as its neighbour where the error reaches a border; the second product's sums as the first one's;
    ``result_eps`` for the rounding of every expert's result, and of the sum."""
    rows = stands_for(x.double())
    out = torch.zeros_like(rows)
    total = torch.zeros_like(rows)
    for e in range(up.shape[0]):
        token, choice = torch.nonzero(chosen == e, as_tuple=True)
        if not token.numel():
            continue
        y, dy = activated(rows[token], up[e], kind, gated, params)
        held, off = stands_for(y), moved(y, dy)
        z = held @ down[e].T
        dz = off @ down[e].abs().T + ((held.abs() + off) @ down[e].abs().T) * (y.shape[1] / 32 + 4) * 2.0 ** -24
        share = weights[token, choice].double()[:, None]
        out.index_add_(0, token, share * (dz + (z.abs() + dz) * result_eps))
        total.index_add_(0, token, share * z.abs())
    return out + total * 2.0 ** -22 + (total + out) * result_eps
