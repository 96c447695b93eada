"""Cases of the operators around weights in 8 bits: bringing rows to 8 bits, products of such rows with such weights, experts of them.

``rows``     rows of numbers become 8-bit rows: as they are, behind a residual sum and an RMS norm, or behind a gated activation.
``product``  ``x @ w.T`` of 8-bit rows (or of bfloat16 rows, which the call brings to 8 bits first) and an 8-bit weight.
``experts``  a feed-forward of routed experts with 8-bit weights: every token through its chosen experts, weighted and added up.

How rows are held.  A row of ``K`` numbers (``K`` a multiple of 16) is ``K`` numbers of E4M3 and a scale, a power of two, for every 128
neighbouring ones: ``codes`` ``[rows, K]`` (float8_e4m3fn) and ``scales`` ``[rows, 4 * ceil(K / 512)]`` (float8_e8m0fnu, the places
behind ``ceil(K / 128)`` hold byte 0).  The scale of 128 numbers with largest finite magnitude ``a`` is ``2 ** e``, ``e`` the least integer
with ``a <= 448 * 2 ** e``, at least -126 and at most 120 (-126 where ``a`` is 0); a number is divided by it and rounded to nearest, ties to
even; what is not finite becomes NaN.  A weight ``[N, K]`` is ``N`` such rows, the weights of ``E`` experts are ``[E, N, K]``.
"""

from __future__ import annotations

import math
import random
from typing import Dict, List, Optional, Tuple

import torch

own = False

BLOCK = 128          # numbers that share a scale
TOP = 448.0          # the largest number of E4M3
EPS = 1e-5


def _rows(name: str, form: str, tokens: int, width: int, dtype: str = "bfloat16") -> dict:
    return dict(name=name, kind="rows", form=form, tokens=tokens, width=width, dtype=dtype)


def _product(name: str, tokens: int, out: int, width: int, rows: str = "fp8") -> dict:
    return dict(name=name, kind="product", tokens=tokens, out=out, width=width, rows=rows)


def _experts(name: str, tokens: int, experts: int, top: int, width: int, hidden: int, gated: bool) -> dict:
    return dict(name=name, kind="experts", tokens=tokens, experts=experts, top=top, width=width, hidden=hidden, gated=gated)


def listed() -> List[dict]:
    # widths of the framework's 1B (2,048 / 8,192) and 8B (4,096 / 14,336) shapes and of its benchmark's layers of experts
    return [
        # one user's decoded token on the small shape, what attention left of it: the smallest call
        _rows("rows_token", "plain", 1, 2048),
        # a decode step of eight requests: a sublayer's result onto the stream, then the next norm
        _rows("norm_8", "norm", 8, 4096),
        # the same for a prompt being read
        _rows("norm_prompt", "norm", 2048, 4096),
        # a portion of odd length behind the gate and up products of the large shape
        _rows("gate_portion", "gate", 1531, 14336),
        # 32-bit rows, a width whose last scale has 48 numbers only
        _rows("rows_f32_odd", "plain", 777, 5040, "float32"),
        # one decoded token of the large shape leaves attention: rows in bfloat16
        _product("decode_1", 1, 4096, 4096, "bfloat16"),
        # the benchmark's headline, eight requests: the stacked gate and up weight
        _product("decode_8", 8, 28672, 4096),
        # a full batch: the down product
        _product("decode_64", 64, 4096, 14336),
        # portions of odd length on the small shape
        _product("portion_odd", 701, 2048, 8192, "bfloat16"),
        # a prompt through the stacked gate and up weight
        _product("prompt_2048", 2048, 28672, 4096),
        # eight decoded tokens through the benchmark's large layer of experts
        _experts("experts_8", 8, 32, 4, 4096, 3584, False),
        # a prompt through it, with gated experts
        _experts("experts_prompt", 2048, 32, 4, 4096, 3584, True),
    ]


def _log(rng, lo: int, hi: int) -> int:
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _sixteens(rng, lo: int, hi: int) -> int:
    return 16 * _log(rng, lo // 16, hi // 16)


def draw(rng) -> dict:
    u = rng.random()
    if u < 0.35:
        form = rng.choice(["plain", "norm", "gate"])
        width = rng.choice([2048, 4096, 8192, 14336]) if rng.random() < 0.5 else _sixteens(rng, 64, 16384)
        case = _rows("", form, _log(rng, 1, 3000), width, "float32" if rng.random() < 0.3 else "bfloat16")
    elif u < 0.75:
        width = rng.choice([2048, 4096, 8192, 14336]) if rng.random() < 0.6 else _sixteens(rng, 64, 14336)
        out = rng.choice([2048, 4096, 6144, 16384, 28672]) if rng.random() < 0.6 else _log(rng, 64, 28672)
        tokens = _log(rng, 1, 64) if rng.random() < 0.5 else _log(rng, 65, 2048)
        while tokens * out * width > 2048 * 28672 * 4096:
            tokens = tokens * 3 // 4
        case = _product("", tokens, out, width, rng.choice(["fp8", "bfloat16"]))
    else:
        experts = rng.choice([8, 16, 32, 64])
        top = rng.choice([1, 2, 4, 8])
        width = rng.choice([2048, 4096]) if rng.random() < 0.6 else _sixteens(rng, 256, 4096)
        hidden = _sixteens(rng, 128, 3584 if experts <= 32 else 2048)
        tokens = _log(rng, 1, 2048)
        while tokens * top * width * hidden > 2048 * 4 * 4096 * 3584:
            tokens = tokens * 3 // 4
        case = _experts("", tokens, experts, top, width, hidden, rng.random() < 0.5)
    del case["name"]
    return case


# ------------------------------------------------------------------------------------------------- sizes of a case

def _held(rows: float, width: int) -> float:
    """Bytes of so many 8-bit rows."""
    return rows * (width + -(-width // BLOCK))


def work(case: dict) -> Dict[str, float]:
    T, K = case["tokens"], case["width"]
    if case["kind"] == "rows":
        size = 4 if case["dtype"] == "float32" else 2
        form = case["form"]
        read = {"plain": T * K * size, "norm": T * K * (8 + size) + 4 * K, "gate": 2 * T * K * size}[form]
        return {"bytes": float(read + _held(T, K)), "flops": float(T * K * {"plain": 2, "norm": 6, "gate": 7}[form])}
    if case["kind"] == "product":
        N = case["out"]
        rows = _held(T, K) if case["rows"] == "fp8" else 2.0 * T * K
        return {"bytes": float(rows + _held(N, K) + 2 * T * N), "flops": float(2 * T * N * K)}
    E, top, hidden = case["experts"], case["top"], case["hidden"]
    up = hidden * (2 if case["gated"] else 1)
    reached = E * (1.0 - (1.0 - top / E) ** T)           # experts that some token chooses, were all alike
    weights = reached * (_held(up, K) + _held(K, hidden))
    return {"bytes": float(weights + 4 * T * K + 8 * T * top), "flops": float(2 * T * top * K * (up + hidden))}


# ------------------------------------------------------------------------------------------------- the plain forms

def _blocks(x: torch.Tensor) -> torch.Tensor:
    """``[..., K]`` -> ``[..., ceil(K / 128), 128]``, zeros behind the last column."""
    pad = -x.shape[-1] % BLOCK
    return torch.nn.functional.pad(x, (0, pad)).unflatten(-1, (-1, BLOCK))


def _encode(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """float32 ``[..., K]`` -> codes ``[..., K]`` and scales ``[..., 4 * ceil(K / 512)]``."""
    g = _blocks(x)
    fine = torch.isfinite(g)
    top = torch.where(fine, g.abs(), torch.zeros_like(g)).amax(-1)
    part, power = torch.frexp(top)                                      # top = part * 2 ** power, part below 1
    e = torch.where(part <= TOP / 512.0, power - 9, power - 8).clamp(-126, 120)
    e = torch.where(top == 0, torch.full_like(e, -126), e)
    byte = (e + 127).to(torch.uint8)
    scale = byte.view(torch.float8_e8m0fnu).float()[..., None]
    codes = torch.where(fine, g / scale, torch.full_like(g, math.nan)).to(torch.float8_e4m3fn)
    scales = torch.nn.functional.pad(byte, (0, -e.shape[-1] % 4)).view(torch.float8_e8m0fnu)
    return codes.flatten(-2)[..., :x.shape[-1]].contiguous(), scales


def _decode(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """What 8-bit rows stand for, float32."""
    K = codes.shape[-1]
    n = -(-K // BLOCK)
    return (_blocks(codes.float()) * scales[..., :n].float()[..., None]).flatten(-2)[..., :K]


def _gate(u: torch.Tensor) -> torch.Tensor:
    g, up = u.chunk(2, -1)
    return g / (1.0 + torch.exp(-g)) * up


def _plain_rows(s: dict):
    if s["form"] == "norm":
        s["h"].add_(s["delta"].float())
        y = s["h"] * torch.rsqrt((s["h"] * s["h"]).mean(-1, keepdim=True) + EPS) * s["weight"]
        codes, scales = _encode(y)
        return {"h": s["h"], "codes": codes, "scales": scales}
    x = s["x"].float()
    codes, scales = _encode(_gate(x) if s["form"] == "gate" else x)
    return {"codes": codes, "scales": scales}


def _plain_product(s: dict):
    x = (s["x"], s["x_scales"]) if "x_scales" in s else _encode(s["x"].float())
    return torch.matmul(_decode(*x), _decode(s["w"], s["w_scales"]).T).to(torch.bfloat16)


def _plain_experts(s: dict):
    """The (token, choice) pairs, sorted by expert, in chunks of one expert each; a chunk's rows times its expert's matrices."""
    T, top = s["chosen"].shape
    E, pairs = s["up"].shape[0], T * top
    size = 64 if pairs > 1024 else 8
    expert, order = torch.sort(s["chosen"].reshape(-1).long(), stable=True)
    count = (expert[:, None] == torch.arange(E, device=expert.device)).sum(0)
    chunks = (count + size - 1) // size
    first_chunk, first = chunks.cumsum(0) - chunks, count.cumsum(0) - count
    place = first_chunk[expert] * size + torch.arange(pairs, device=expert.device) - first[expert]
    n = min(pairs, E + pairs // size)                     # as many chunks as there can be
    of_chunk = (torch.arange(n, device=expert.device)[:, None] >= (first_chunk + chunks)).sum(-1).clamp(max=E - 1)
    x = _decode(*_encode(s["x"].float()))
    rows = torch.zeros((n * size, x.shape[1]), device=x.device)
    rows[place] = x[order // top]
    u = torch.matmul(rows.reshape(n, size, -1), _decode(s["up"][of_chunk], s["up_scales"][of_chunk]).transpose(1, 2))
    u = _gate(u) if s["gated"] else torch.relu(u) ** 2
    y = torch.matmul(_decode(*_encode(u)), _decode(s["down"][of_chunk], s["down_scales"][of_chunk]).transpose(1, 2))
    out = torch.zeros((pairs, x.shape[1]), device=x.device)
    out[order] = y.reshape(n * size, -1)[place]
    return (out.reshape(T, top, -1) * s["share"][..., None]).sum(1).to(torch.bfloat16)


# ------------------------------------------------------------------------------------------------- a pass

def _dtype(name: str) -> torch.dtype:
    return torch.float32 if name == "float32" else torch.bfloat16


def prepare(case: dict, seed: int) -> dict:
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    randn = lambda *shape: torch.randn(shape, generator=gen, device="cuda")  # noqa: E731
    T, K = case["tokens"], case["width"]
    # some channels of activations are far larger than others
    gain = torch.exp(0.5 * randn(K))
    gain = torch.where(torch.rand(K, generator=gen, device="cuda") < 0.01, 12.0 * gain, gain)
    state: dict = {"kind": case["kind"]}
    if case["kind"] == "rows":
        dtype = _dtype(case["dtype"])
        state["form"] = case["form"]
        if case["form"] == "norm":
            state.update(h=randn(T, K) * gain * 3.0, delta=(randn(T, K) * 0.3).to(dtype), weight=1.0 + 0.2 * randn(K))
        elif case["form"] == "gate":
            state["x"] = (randn(T, 2 * K) * torch.cat([gain, gain])).to(dtype)
        else:
            state["x"] = (randn(T, K) * gain).to(dtype)
    elif case["kind"] == "product":
        x = randn(T, K) * gain
        if case["rows"] == "fp8":
            state["x"], state["x_scales"] = _encode(x)
        else:
            state["x"] = x.to(torch.bfloat16)
        # rows of weights are of different sizes
        state["w"], state["w_scales"] = _encode(randn(case["out"], K) * (K ** -0.5 * torch.exp(0.3 * randn(case["out"], 1))))
    else:
        E, top, hidden = case["experts"], case["top"], case["hidden"]
        up = hidden * (2 if case["gated"] else 1)
        state.update(gated=case["gated"], x=(randn(T, K) * gain).to(torch.bfloat16))
        state["up"], state["up_scales"] = _encode(randn(E, up, K) * K ** -0.5)
        state["down"], state["down_scales"] = _encode(randn(E, K, hidden) * hidden ** -0.5)
        score = randn(T, E) + 0.7 * randn(E)              # some experts are chosen more often than others
        best, chosen = torch.topk(score, top, dim=-1)
        state.update(chosen=chosen.int().contiguous(), share=torch.softmax(best, -1).contiguous())
    if own:
        from torchllms_b200.kernels import get_ops
        from torchllms_b200.weights.fp8 import Fp8Rows
        state.update(ops=get_ops(), held={k: Fp8Rows(state[k], state[k + "_scales"]) for k in ("x", "w", "up", "down") if k + "_scales" in state})
    return state


def run(s: dict):
    if not own:
        return {"rows": _plain_rows, "product": _plain_product, "experts": _plain_experts}[s["kind"]](s)
    ops, held = s["ops"], s["held"]
    if s["kind"] == "product":
        return ops.linear_fp8(held["x"] if "x" in held else s["x"], held["w"])
    if s["kind"] == "experts":
        return ops.moe_experts_fp8(s["x"], s["chosen"], s["share"], held["up"], held["down"], activation="silu" if s["gated"] else "relu2",
                                   gated=s["gated"])
    if s["form"] == "norm":
        rows = ops.rmsnorm_fp8(s["h"], s["delta"], s["weight"], EPS)
        return {"h": s["h"], "codes": rows.codes, "scales": rows.scales}
    rows = ops.activation_fp8(s["x"], "silu", gated=True) if s["form"] == "gate" else ops.quantize_fp8(s["x"])
    return {"codes": rows.codes, "scales": rows.scales}


# ------------------------------------------------------------------------------------------------- in 64 bits

def _exact_rows(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """64-bit ``[rows, K]``: the numbers that are held (before their scale), ``[rows, K]``, and the scale of every 128, by the definition."""
    R, K = x.shape
    n = -(-K // BLOCK)
    g = torch.zeros((R, n * BLOCK), dtype=torch.float64, device=x.device)
    g[:, :K] = x
    g = g.reshape(R, n, BLOCK)
    a = g.abs().amax(-1, keepdim=True)
    e = torch.ceil(torch.log2((a / TOP).clamp(min=2.0 ** -126)))
    e = torch.where(a > TOP * torch.exp2(e), e + 1, torch.where((a <= TOP * torch.exp2(e - 1)) & (e > -126), e - 1, e))
    v = g / torch.exp2(e)
    quantum = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6))) - 3)
    return ((v / quantum).round() * quantum).flatten(1)[:, :K], torch.exp2(e[..., 0])


def _exact_value(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    K = codes.shape[-1]
    return codes.double() * scales.double().repeat_interleave(BLOCK, -1)[..., :K]


def _stands_for(x: torch.Tensor) -> torch.Tensor:
    return _exact_value(*_exact_rows(x))


def exact(case: dict, seed: int) -> Optional[object]:
    s = prepare(case, seed)
    if case["kind"] == "product":
        x = _exact_value(s["x"], s["x_scales"]) if case["rows"] == "fp8" else _stands_for(s["x"].double())
        return x @ _exact_value(s["w"], s["w_scales"]).T
    silu = torch.nn.functional.silu
    if case["kind"] == "rows":
        K = case["width"]
        if case["form"] == "norm":
            h = s["h"].double() + s["delta"].double()
            y = h / torch.sqrt(h.pow(2).sum(-1, keepdim=True) / K + EPS) * s["weight"].double()
        elif case["form"] == "gate":
            x = s["x"].double()
            y = silu(x[:, :K]) * x[:, K:]
        else:
            y = s["x"].double()
        codes, scale = _exact_rows(y)
        scales = torch.full((y.shape[0], 4 * -(-K // 512)), 2.0 ** -127, dtype=torch.float64, device=y.device)
        scales[:, :scale.shape[1]] = scale
        return {"h": h, "codes": codes, "scales": scales} if case["form"] == "norm" else {"codes": codes, "scales": scales}
    x, hidden = _stands_for(s["x"].double()), case["hidden"]
    out = torch.zeros_like(x)
    for e in range(case["experts"]):
        token, choice = torch.nonzero(s["chosen"] == e, as_tuple=True)
        u = x[token] @ _exact_value(s["up"][e], s["up_scales"][e]).T
        u = silu(u[:, :hidden]) * u[:, hidden:] if case["gated"] else u.clamp(min=0) ** 2
        y = _stands_for(u) @ _exact_value(s["down"][e], s["down_scales"][e]).T
        out.index_add_(0, token, y * s["share"][token, choice].double()[:, None])
    return out
