"""Cases of the operators around a cache of keys and values held in 4 bits: writing it and attending over it.

``append``     the step's projected rows are rotated, q leaves as it is, k and v go to their places in the paged cache as
               4-bit numbers with an 8-bit scale for 16 of them; then the values that the cache now stands for are read
               back, of the tokens written and of earlier ones beside them.
``attention``  grouped-query attention of the step's queries over such a cache: causal, over pages in any order, with or
               without a window, for requests that bring one token each, a few, or portions of their prompts.

How the cache is laid out.  Sixteen tokens of one key head are a record of ``9 * dim`` bytes: 16 rows of ``dim / 2`` bytes,
coordinate ``2 i`` in the low and ``2 i + 1`` in the high half of byte ``i``, then 16 rows of ``dim / 16`` scales, a byte for 16
neighbouring coordinates.  Pages are ``[page, kv_head, page_size / 16, 9 * dim]``, uint8.  A 4-bit number is a sign and one of
0, 0.5, 1, 1.5, 2, 3, 4, 6 (E2M1); a scale is 5 bits of exponent and 3 of mantissa without a sign (bias 15, subnormal below
2^-14).  Of 16 numbers with largest magnitude ``a`` the scale is ``a / 6``, rounded to nearest (ties to even) and at most 10240;
a number is divided by the scale and rounded to nearest, ties to the even code, at most 6.
"""

from __future__ import annotations

import math
import random
from typing import Dict, List, Optional, Tuple

import torch

own = False

GROUP = 16           # numbers that share a scale
RECORD = 16          # tokens of a record
TOP_SCALE = 226      # the scale byte of 10240


def _case(name: str, kind: str, dtype: str = "bfloat16", heads: int = 32, kv_heads: int = 8, dim: int = 128, page: int = 16,
          requests: int = 1, new: Tuple[int, int] = (1, 1), behind: Tuple[int, int] = (0, 0), window: int = 0, rotated: int = 0,
          pairing: str = "interleaved", lengths: int = 0) -> dict:
    """``requests`` bring ``new`` (least, most) tokens each behind ``behind`` (least, most) earlier ones; ``lengths`` says which."""
    case = dict(name=name, kind=kind, dtype=dtype, heads=heads, kv_heads=kv_heads, dim=dim, page=page, requests=requests, new_lo=new[0],
                new_hi=new[1], behind_lo=behind[0], behind_hi=behind[1], lengths=lengths)
    if kind == "append":
        case.update(rotated=rotated or dim, pairing=pairing)
    else:
        case.update(window=window)
    return case


def listed() -> List[dict]:
    # heads as the framework's 1B (32 / 8 of 64) and 8B (32 / 8 of 128) shapes have them
    return [
        # the smallest call: one user's decoded token goes into the cache
        _case("append_token", "append", dim=64, behind=(332, 332)),
        # a step that reads prompts: portions of several requests at once
        _case("append_portions", "append", requests=5, new=(700, 2400), behind=(0, 3000), lengths=1),
        # 32 bits, halves of the rotated part paired, a part of the head passes unrotated; odd numbers of tokens
        _case("append_f32", "append", "float32", requests=3, new=(101, 333), behind=(1, 90), rotated=64, pairing="half", page=64, lengths=2),
        # one user talking to a small model: latency
        _case("decode_1", "attention", dim=64, behind=(332, 332)),
        # the headline of the framework's benchmark: eight requests behind prompts of 2,048
        _case("decode_8", "attention", requests=8, behind=(2048, 2048)),
        # a full batch of requests of all lengths
        _case("decode_64", "attention", requests=64, behind=(200, 16000), lengths=3),
        # few requests deep into long documents, what a 4-bit cache is for; larger pages
        _case("decode_long", "attention", requests=4, behind=(27001, 32767), page=64, lengths=4),
        # 32-bit decoding, several tokens at a time (a draft being checked), inside a window
        _case("draft_f32_window", "attention", "float32", dim=64, requests=12, new=(2, 4), behind=(90, 3900), window=1024, lengths=5),
        # a whole prompt at once
        _case("prompt_2048", "attention", new=(2048, 2048)),
        # a long document being read: a portion behind what was read before
        _case("portion_far", "attention", new=(2048, 2048), behind=(14001, 14001), page=64),
        # portions of odd lengths of several requests on the small shape
        _case("portions_odd", "attention", dim=64, requests=6, new=(70, 1100), behind=(0, 2500), lengths=6),
        # 32-bit scoring of a prompt
        _case("prompt_f32", "attention", "float32", dim=64, requests=2, new=(500, 901), lengths=7),
    ]


def _log(rng, lo: int, hi: int) -> int:
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng) -> dict:
    dtype = "float32" if rng.random() < 0.25 else "bfloat16"
    heads, kv_heads, dim = rng.choice([(32, 8, 64), (32, 8, 128), (32, 8, 128), (16, 16, 64), (64, 8, 128), (8, 1, 128), (28, 4, 128)])
    page = rng.choice([16, 16, 32, 64, 128])
    lengths = rng.randrange(1 << 20)
    u = rng.random()
    if u < 0.25:
        requests = _log(rng, 1, 64)
        most = 1 if rng.random() < 0.4 else _log(rng, 2, max(2, 9000 // requests))
        case = _case("", "append", dtype, heads, kv_heads, dim, page, requests, (_log(rng, 1, most), most), (0, _log(rng, 1, 4000)),
                     rotated=rng.choice([dim, dim, dim // 2]), pairing=rng.choice(["interleaved", "half"]), lengths=lengths)
    elif u < 0.65:
        requests = _log(rng, 1, 64)
        far = _log(rng, 17, min(32000, 380_000 // requests))
        most = rng.choice([1, 1, 1, 2, 4])
        case = _case("", "attention", dtype, heads, kv_heads, dim, page, requests, (1, most), (_log(rng, 1, far), far),
                     window=_log(rng, 64, 4096) if rng.random() < 0.2 else 0, lengths=lengths)
    else:
        requests = rng.choice([1, 1, 2, 3, 6])
        most = _log(rng, 5, 4000 // requests)
        far = 0 if rng.random() < 0.4 else _log(rng, 9, 12000 // requests)
        while heads * requests * most * (most + far) > 32 * 2048 * 12000:      # (a plain form's scores)
            most, far = most * 3 // 4, far * 3 // 4
        case = _case("", "attention", dtype, heads, kv_heads, dim, page, requests, (_log(rng, 2, most), most), (0, far),
                     window=_log(rng, 64, 4096) if rng.random() < 0.2 else 0, lengths=lengths)
    del case["name"]
    return case


# ------------------------------------------------------------------------------------------------- sizes of a case

def _sizes(case: dict) -> Tuple[List[int], List[int]]:
    """New tokens and earlier tokens of every request."""
    rng = random.Random(case["lengths"])
    spread = lambda lo, hi: hi if lo >= hi else rng.randint(lo, hi)  # noqa: E731
    new = [spread(case["new_lo"], case["new_hi"]) for _ in range(case["requests"])]
    behind = [spread(case["behind_lo"], case["behind_hi"]) for _ in range(case["requests"])]
    return new, behind


def _read_back(case: dict, new: List[int], behind: List[int]) -> List[Tuple[int, int]]:
    """(request, position) of the tokens that ``append`` reads back: all new ones, and up to 16 earlier ones of every request."""
    return [(b, t) for b, (n, s) in enumerate(zip(new, behind)) for t in range(max(0, s - 16), s + n)]


def work(case: dict) -> Dict[str, float]:
    new, behind = _sizes(case)
    H, KV, D = case["heads"], case["kv_heads"], case["dim"]
    size = 4 if case["dtype"] == "float32" else 2
    T, token = sum(new), 2 * KV * (D // 2 + D // GROUP)        # bytes of a token in the cache
    if case["kind"] == "append":
        back = len(_read_back(case, new, behind))
        moved = T * (H + 2 * KV) * D * size + T * H * D * size + T * token + T * 4 * case["rotated"] + back * (token + 2 * KV * D * size)
        return {"bytes": float(moved), "flops": float(T * ((H + KV) * case["rotated"] * 3 + 2 * KV * D * 2))}
    window = case["window"] or (1 << 40)
    keys = sum(min(s + n, n + window - 1) for n, s in zip(new, behind))
    pairs = sum(min(s + i + 1, window) for n, s in zip(new, behind) for i in range(n))
    return {"bytes": float(2 * T * H * D * size + keys * token), "flops": float(4 * pairs * H * D)}


# ------------------------------------------------------------------------------------------------- the plain forms

def _tables(device) -> Tuple[torch.Tensor, torch.Tensor]:
    """The two numbers of every byte, and the scale of every byte."""
    magnitude = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=device)
    numbers = torch.cat([magnitude, -magnitude])
    byte = torch.arange(256, device=device)
    exponent, mantissa = byte >> 3, (byte & 7).float()
    scale = torch.where(exponent == 0, mantissa * 2.0 ** -17, (8.0 + mantissa) * torch.exp2((exponent - 18).float()))
    return torch.stack([numbers[byte & 15], numbers[byte >> 4]], dim=1), scale


def _decode(records: torch.Tensor, D: int) -> torch.Tensor:
    """Records ``[..., 9 D]`` -> the numbers they stand for, float32 ``[..., 16, D]``."""
    pairs, scale = _tables(records.device)
    codes, scales = records[..., :8 * D].reshape(-1, D // 16, 8), records[..., 8 * D:].reshape(-1, D // 16)
    values = pairs[codes.int()].reshape(-1, D // 16, GROUP) * scale[scales.int()][..., None]
    return values.reshape(*records.shape[:-1], RECORD, D)


def _encode(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """float32 ``[..., D]`` -> bytes of 4-bit numbers ``[..., D / 2]`` and of scales ``[..., D / 16]``."""
    groups = x.reshape(*x.shape[:-1], -1, GROUP)
    wanted = groups.abs().amax(-1) / torch.full((), 6.0, device=x.device)
    bits = wanted.view(torch.int32)
    normal = ((bits + 0x7FFFF + ((bits >> 20) & 1)) >> 20) - (112 << 3)
    scales = torch.where(wanted < 2.0 ** -14, (wanted * 2.0 ** 17).round().int(), normal).clamp(max=TOP_SCALE)
    scale = _tables(x.device)[1][scales][..., None]
    a = torch.where(scale > 0, groups.abs() / scale, torch.zeros_like(groups))
    code = ((a > 0.25).int() + (a >= 0.75).int() + (a > 1.25).int() + (a >= 1.75).int() + (a > 2.5).int() + (a >= 3.5).int() + (a > 5.0).int())
    code = torch.where(groups < 0, code + 8, code).reshape(*x.shape[:-1], -1, 2)
    return (code[..., 0] + 16 * code[..., 1]).to(torch.uint8), scales.to(torch.uint8)


def _rotate(x: torch.Tensor, cs: torch.Tensor, pairing: str) -> torch.Tensor:
    """The first ``2 * cs.shape[-2]`` coordinates of ``x`` ``[T, heads, D]`` by the angles whose (cos, sin) are ``cs`` ``[T, 1, pairs, 2]``."""
    n = 2 * cs.shape[-2]
    c, s = cs[..., 0], cs[..., 1]
    x0, x1 = (x[..., 0:n:2], x[..., 1:n:2]) if pairing == "interleaved" else (x[..., :n // 2], x[..., n // 2:n])
    y0, y1 = x0 * c - x1 * s, x1 * c + x0 * s
    y = torch.stack([y0, y1], -1).flatten(-2) if pairing == "interleaved" else torch.cat([y0, y1], -1)
    return torch.cat([y, x[..., n:]], -1)


def _record_of(slots: torch.Tensor, page: int) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    return slots // page, slots % page // RECORD, slots % RECORD


def _plain_store(pages: torch.Tensor, x: torch.Tensor, slots: torch.Tensor, page: int) -> None:
    """Numbers ``x`` ``[T, KV, D]`` into their places."""
    D = x.shape[-1]
    codes, scales = _encode(x)
    p, r, i = _record_of(slots.long(), page)
    pages[..., :8 * D].unflatten(-1, (RECORD, D // 2))[p, :, r, i] = codes
    pages[..., 8 * D:].unflatten(-1, (RECORD, D // GROUP))[p, :, r, i] = scales


def _plain_load(pages: torch.Tensor, slots: torch.Tensor, page: int, D: int) -> torch.Tensor:
    """The numbers of these places, ``[n, KV, D]``."""
    p, r, i = _record_of(slots.long(), page)
    codes = pages[..., :8 * D].unflatten(-1, (RECORD, D // 2))[p, :, r, i]
    scales = pages[..., 8 * D:].unflatten(-1, (RECORD, D // GROUP))[p, :, r, i]
    pairs, scale = _tables(pages.device)
    return (pairs[codes.int()].reshape(*codes.shape[:2], -1, GROUP) * scale[scales.int()][..., None]).flatten(2)


def _plain_append(s: dict):
    x = s["qkv"].float().unflatten(1, (-1, s["D"]))
    cs = s["table"][s["positions"].long()][:, None]
    H, KV = s["H"], s["KV"]
    turned = _rotate(x[:, :H + KV], cs, s["pairing"])
    _plain_store(s["k_pages"], turned[:, H:], s["slots"], s["page"])
    _plain_store(s["v_pages"], x[:, H + KV:], s["slots"], s["page"])
    read = [_plain_load(pages, s["read"], s["page"], s["D"]).to(s["dtype"]) for pages in (s["k_pages"], s["v_pages"])]
    return {"q": turned[:, :H].to(s["dtype"]), "k": read[0], "v": read[1]}


def _plain_attention(s: dict):
    H, KV, D, page = s["H"], s["KV"], s["D"], s["page"]
    q_start, kv_len, q = s["q_start"].long(), s["kv_len"].long(), s["q"].float()
    B, most = kv_len.numel(), s["max_q_len"]
    new = q_start[1:] - q_start[:-1]
    step = torch.arange(most, device=q.device)
    there = step < new[:, None]                                                            # [B, most]
    rows = torch.where(there, q_start[:-1, None] + step, torch.zeros_like(there, dtype=torch.long))
    padded = q[rows].reshape(B, most, KV, H // KV, D).permute(0, 2, 3, 1, 4).reshape(B, KV, -1, D)
    table = s["block_table"].long().clamp(min=0)
    gather = lambda pages: _decode(pages[table], D).permute(0, 2, 1, 3, 4, 5).reshape(B, KV, -1, D)  # noqa: E731
    scores = (torch.matmul(padded, gather(s["k_pages"]).transpose(2, 3)) * s["scale"]).reshape(B, KV, H // KV, most, -1)
    key = torch.arange(scores.shape[-1], device=q.device)
    at = (kv_len - new)[:, None] + step                                                    # positions of the queries
    seen = (key <= at[..., None]) & there[..., None] & (key < kv_len[:, None, None])
    if s["window"]:
        seen = seen & (key > at[..., None] - s["window"])
    seen = seen[:, None, None]
    scores = scores.masked_fill(~seen, -math.inf)
    top = scores.amax(-1, keepdim=True)
    weight = torch.exp(scores - top.masked_fill(top == -math.inf, 0.0))
    total = weight.sum(-1, keepdim=True)
    out = torch.matmul(weight.reshape(B, KV, -1, key.numel()), gather(s["v_pages"])).reshape(B, KV, H // KV, most, D)
    out = (out / total.masked_fill(total == 0.0, 1.0)).permute(0, 3, 1, 2, 4).reshape(B, most, H, D)
    return out[there].to(s["dtype"])


# ------------------------------------------------------------------------------------------------- a pass

def _numbers(gen, shape, gain: torch.Tensor) -> torch.Tensor:
    return torch.randn(shape, generator=gen, device="cuda") * gain


def prepare(case: dict, seed: int) -> dict:
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    host = random.Random(seed)
    new, behind = _sizes(case)
    H, KV, D, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    dtype = torch.float32 if case["dtype"] == "float32" else torch.bfloat16
    blocks = [-(-(n + s) // page) for n, s in zip(new, behind)]
    order = list(range(sum(blocks) + 3))                  # (three pages are nobody's)
    host.shuffle(order)
    table, at = [], 0
    for n in blocks:
        table.append(order[at:at + n] + [-1] * (max(blocks) - n))
        at += n
    ints = lambda v: torch.tensor(v, dtype=torch.int32).cuda()  # noqa: E731
    # what the cache holds: some channels of the keys are far larger than others, values are even
    gain = torch.exp(0.4 * torch.randn((KV, 1, D), generator=gen, device="cuda"))
    gain = torch.where(torch.rand((KV, 1, D), generator=gen, device="cuda") < 0.03, 4.0 * gain, gain)
    records = (len(order), KV, page // RECORD)
    pages = []
    for g in (gain, torch.full_like(gain, 0.6)):
        codes, scales = _encode(_numbers(gen, (*records[:2], page, D), g))
        pages.append(torch.cat([codes.reshape(*records, -1), scales.reshape(*records, -1)], -1).contiguous())
    state = dict(kind=case["kind"], H=H, KV=KV, D=D, page=page, dtype=dtype, k_pages=pages[0], v_pages=pages[1])
    slot = lambda b, t: table[b][t // page] * page + t % page  # noqa: E731
    if case["kind"] == "append":
        rotated = case["rotated"]
        angle = torch.arange(max(behind) + max(new), device="cuda", dtype=torch.float64)[:, None] * 5e5 ** (
            -torch.arange(0, rotated, 2, device="cuda", dtype=torch.float64) / rotated)
        state.update(table=torch.stack([angle.cos(), angle.sin()], -1).float().contiguous(), pairing=case["pairing"],
                     positions=ints([s + i for n, s in zip(new, behind) for i in range(n)]),
                     slots=ints([slot(b, s + i) for b, (n, s) in enumerate(zip(new, behind)) for i in range(n)]),
                     read=ints([slot(b, t) for b, t in _read_back(case, new, behind)]))
        gains = torch.cat([torch.ones((H, D), device="cuda"), gain[:, 0], torch.full((KV, D), 0.6, device="cuda")])
        state["qkv"] = _numbers(gen, (sum(new), (H + 2 * KV) * D), gains.reshape(-1)).to(dtype)
    else:
        starts = [sum(new[:b]) for b in range(len(new) + 1)]
        sharp = torch.linspace(0.4, 2.0, H, device="cuda")[:, None]      # heads look at many keys, or at few
        state.update(q=_numbers(gen, (sum(new), H, D), sharp).to(dtype), block_table=ints(table), q_start=ints(starts),
                     kv_len=ints([n + s for n, s in zip(new, behind)]), max_q_len=max(new), max_kv_len=max(n + s for n, s in zip(new, behind)),
                     window=case["window"] or None, scale=D ** -0.5)
    if own:
        from torchllms_b200.kernels import get_ops
        state["ops"] = get_ops()
    return state


def run(s: dict):
    if not own:
        return _plain_append(s) if s["kind"] == "append" else _plain_attention(s)
    ops = s["ops"]
    if s["kind"] == "append":
        q = ops.rope_kv_write_fp4(s["qkv"], s["positions"], s["table"], n_heads=s["H"], n_kv_heads=s["KV"], head_dim=s["D"],
                                  interleaved=s["pairing"] == "interleaved", k_pages=s["k_pages"], v_pages=s["v_pages"],
                                  slot_mapping=s["slots"], page_size=s["page"])
        k, v = ops.kv_read_fp4(s["k_pages"], s["v_pages"], s["read"], head_dim=s["D"], page_size=s["page"], out_dtype=s["dtype"])
        return {"q": q, "k": k, "v": v}
    return ops.paged_attention_fp4(s["q"], s["k_pages"], s["v_pages"], s["block_table"], s["q_start"], s["kv_len"],
                                   n_seqs=s["kv_len"].numel(), max_q_len=s["max_q_len"], max_kv_len=s["max_kv_len"], scale=s["scale"],
                                   window=s["window"], page_size=s["page"])


# ------------------------------------------------------------------------------------------------- in 64 bits

def _exact_numbers(x: torch.Tensor) -> torch.Tensor:
    """What 64-bit ``x`` ``[..., D]`` becomes in 4 bits, by the definition."""
    g = x.unflatten(-1, (-1, GROUP))
    want = g.abs().amax(-1, keepdim=True) / 6.0
    quantum = torch.exp2(torch.floor(torch.log2(want.clamp(min=2.0 ** -14))) - 3.0)
    scale = ((want / quantum).round() * quantum).clamp(max=10240.0)
    a = torch.where(scale > 0, g.abs() / scale, torch.zeros_like(g))
    near = torch.where(a < 2.0, (2.0 * a).round() / 2.0, torch.where(a < 4.0, a.round(), 2.0 * (a / 2.0).round())).clamp(max=6.0)
    return (torch.sign(g) * near * scale).flatten(-2)


def _exact_records(records: torch.Tensor, D: int) -> torch.Tensor:
    """Records ``[n, 9 D]`` -> 64-bit numbers ``[16 n, D]``."""
    byte = records[:, :8 * D].reshape(-1, D // 2, 1).long()
    nibble = torch.cat([byte % 16, byte // 16], -1).reshape(-1, D)
    e, m = nibble // 2 % 4, (nibble % 2).double()
    magnitude = torch.where(e == 0, m / 2.0, (1.0 + m / 2.0) * 2.0 ** (e - 1).double())
    s = records[:, 8 * D:].reshape(-1, D // GROUP).long()
    scale = torch.where(s < 8, s.double() * 2.0 ** -17, (1.0 + (s % 8).double() / 8.0) * 2.0 ** (s // 8 - 15).double())
    return torch.where(nibble >= 8, -magnitude, magnitude) * scale.repeat_interleave(GROUP, 1)


def exact(case: dict, seed: int) -> Optional[object]:
    s = prepare(case, seed)
    new, behind = _sizes(case)
    H, KV, D, page = s["H"], s["KV"], s["D"], s["page"]
    if case["kind"] == "append":
        x = s["qkv"].double().reshape(-1, H + 2 * KV, D)
        n, cs = case["rotated"], s["table"].double()[s["positions"].long()]
        first = torch.arange(0, n, 2) if case["pairing"] == "interleaved" else torch.arange(n // 2)
        first = first.cuda()
        second = first + (1 if case["pairing"] == "interleaved" else n // 2)
        y = x[:, :H + KV].clone()
        z = torch.complex(x[:, :H + KV, first], x[:, :H + KV, second]) * torch.complex(cs[..., 0], cs[..., 1])[:, None]
        y[..., first], y[..., second] = z.real, z.imag
        out = {"q": y[:, :H]}
        for name, pages, fresh in (("k", s["k_pages"], y[:, H:]), ("v", s["v_pages"], x[:, H + KV:])):
            old = _exact_records(pages.reshape(-1, 9 * D), D).reshape(-1, KV, page, D)         # [page, KV, slot, D]
            old = old.transpose(1, 2).reshape(-1, KV, D)
            old[s["slots"].long()] = _exact_numbers(fresh)
            out[name] = old[s["read"].long()]
        return out
    outs = []
    for b, (n, before) in enumerate(zip(new, behind)):
        first = int(s["q_start"][b])
        pages = s["block_table"][b, :-(-(n + before) // page)].long()
        at = torch.arange(before, before + n, device="cuda")[:, None]
        key = torch.arange(n + before, device="cuda")[None]
        hidden = (key > at) | (key <= at - (case["window"] or n + before + 1))
        per_head = []
        for h in range(KV):
            k, v = (_exact_records(t[pages, h].reshape(-1, 9 * D), D)[:n + before] for t in (s["k_pages"], s["v_pages"]))
            for g in range(H // KV):
                w = s["q"][first:first + n, h * (H // KV) + g].double() @ k.T * (D ** -0.5)
                per_head.append(torch.softmax(w.masked_fill(hidden, -math.inf), -1) @ v)
        outs.append(torch.stack(per_head, 1))
    return torch.cat(outs)
