"""The 4-bit cache on the host: the format against its definition, pages and needs, the engine over plain twins of the kernels."""

import random

import numpy as np
import pytest
import torch

import fp4_plain
import plain_llama
import traces
from helpers import TINY, tiny_folder
from torch_ops import TorchOps
from torchllms_b200.cache import fp4
from torchllms_b200.cache.manager import CacheManager
from torchllms_b200.parts.base import CacheNeed


class Fp4TorchOps(TorchOps):
    """The plain twins with a 4-bit cache: pages are written and read by ``cache/fp4.py``."""

    def prepare(self, dtype, sampling=True, kv_format="full"):
        pass

    def rope_kv_write_fp4(self, qkv, positions, table, *, n_heads, n_kv_heads, head_dim, interleaved, k_pages, v_pages, slot_mapping,
                          page_size, out_dtype=None):
        T = positions.numel()
        k, v = torch.zeros((T, n_kv_heads, 1, head_dim)), torch.zeros((T, n_kv_heads, 1, head_dim))
        q = self.rope_kv_write(qkv, positions, table, n_heads=n_heads, n_kv_heads=n_kv_heads, head_dim=head_dim, interleaved=interleaved,
                               k_pages=k, v_pages=v, slot_mapping=torch.arange(T), page_size=1, out_dtype=out_dtype)
        fp4.store(k_pages, k[:, :, 0], slot_mapping, page_size)
        fp4.store(v_pages, v[:, :, 0], slot_mapping, page_size)
        return q

    def paged_attention_fp4(self, q, k_pages, v_pages, *args, page_size, **kw):
        k, v = (fp4.decode(*fp4.rows_of(t, q.shape[-1])).flatten(2, 3) for t in (k_pages, v_pages))
        return self.paged_attention(q, k, v, *args, page_size=page_size, **kw)


def numbers(kind: str, shape, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=g)
    if kind == "bfloat16":                      # many quotients lie exactly between two codes
        return x.to(torch.bfloat16).float()
    if kind == "spread":                        # from far below the smallest scale to far beyond the largest
        return x * torch.exp2(torch.randint(-30, 30, (*shape[:-1], 1), generator=g).float())
    if kind == "eighths":                       # ties everywhere
        return torch.randint(-64, 65, shape, generator=g) / 8.0
    return x


@pytest.mark.parametrize("kind", ["normal", "bfloat16", "spread", "eighths"])
def test_encode_is_the_definition(kind):
    x = numbers(kind, (500, 3, 64))
    got = fp4.decode(*fp4.encode(x))
    want = fp4_plain.quantized(x)
    assert torch.equal(got.double(), want)


def test_the_format_holds_what_it_says():
    assert torch.equal(fp4.scale_values("cpu")[:227].double(), fp4_plain.SCALES[:227])
    # a number times its scale is a float16: the kernels multiply exactly what is cached
    products = (fp4_plain.SCALES[:227, None] * fp4_plain.MAGNITUDE).flatten()
    assert torch.equal(products.half().double(), products) and torch.equal(products.to(torch.bfloat16).double(), products)
    # the byte shifted left by 7 is the float16 with the scale's value
    bits = (torch.arange(227, dtype=torch.int16) << 7).view(torch.float16)
    assert torch.equal(bits.double(), fp4_plain.SCALES[:227])
    x = torch.zeros(4, 32)
    x[0, 3], x[1, 20], x[2] = float("inf"), float("nan"), 1e30
    y = fp4.decode(*fp4.encode(x))
    assert y[0, :16].isnan().all() and (y[0, 16:] == 0).all()        # a number that is not finite shows in its group, and only there
    assert y[1, 16:].isnan().all() and (y[1, :16] == 0).all()
    assert (y[2] == 61440.0).all() and (y[3] == 0).all()
    # within a group a number is off by at most the scale (between 4 and 6, or above 6 where the scale was rounded down)
    x = numbers("normal", (1000, 1, 128))
    codes, scales = fp4.encode(x)
    scale = fp4.scale_values("cpu")[scales.long()].repeat_interleave(16, -1)
    assert ((fp4.decode(codes, scales) - x).abs() <= scale).all()


def test_sizes_and_refusals():
    assert fp4.page_shape(5, 2, 48, 64) == (5, 2, 3, 576) and fp4.record_bytes(128) == 1152
    for bad in (8, 24, 0, 272, -16):
        with pytest.raises(ValueError, match="4-bit cache"):
            fp4.page_shape(5, 2, 16, bad)
    for bad in (0, 4, 8, 20):
        with pytest.raises(ValueError, match="pages of a multiple"):
            fp4.page_shape(5, 2, bad, 64)
    with pytest.raises(ValueError, match="cache format"):
        CacheNeed("full", 2, 64, format="fp8")
    with pytest.raises(ValueError, match="one size"):
        CacheNeed("full", 2, 64, v_head_dim=32, format="fp4")
    with pytest.raises(ValueError, match="same vectors"):
        CacheNeed("full", 2, 64).covering(CacheNeed("full", 2, 64, format="fp4"))
    need = CacheNeed("window", 2, 64, 100, format="fp4")
    assert need.covering(CacheNeed("window", 2, 64, 300, format="fp4")) == CacheNeed("window", 2, 64, 300, format="fp4")
    assert need.bytes_per_token(2) == 2 * 2 * 36 and CacheNeed("full", 2, 64).bytes_per_token(2) == 2 * 2 * 64 * 2


def test_manager_lays_out_both_formats_beside_each_other():
    needs = [(CacheNeed("full", 2, 64), None, None), (CacheNeed("full", 2, 64, format="fp4"), None, None),
             (CacheNeed("full", 2, 64, format="fp4"), None, None)]
    m = CacheManager(needs, page_size=16, pool_tokens=64, max_num_seqs=2, max_len=64, dtype=torch.bfloat16, device="cpu")
    assert len(m.groups) == 2 and m.groups[1].k_pages.shape == (2, 4, 2, 1, 576) and m.groups[1].k_pages.dtype == torch.uint8
    assert m.run_view(0, [None, None], [None, None]).format == "full" and m.run_view(2, [None, None], [None, None]).format == "fp4"
    assert m.groups[1].bytes() == 64 * 2 * needs[1][0].bytes_per_token(2)
    with pytest.raises(ValueError, match="pages of a multiple"):
        CacheManager(needs, page_size=8, pool_tokens=64, max_num_seqs=2, max_len=64, dtype=torch.bfloat16, device="cpu")


def test_store_and_load_in_any_order():
    g = torch.Generator().manual_seed(3)
    pages = torch.full(fp4.page_shape(4, 2, 32, 64), 7, dtype=torch.uint8)
    slots = torch.randperm(4 * 32, generator=g)[:50].int()
    x = torch.randn((50, 2, 64), generator=g)
    before = pages.clone()
    fp4.store(pages, x, slots, 32)
    assert torch.equal(fp4.load(pages, slots, 32, 64).double(), fp4_plain.quantized(x))
    rest = torch.tensor([s for s in range(128) if s not in set(slots.tolist())]).int()
    assert torch.equal(fp4.load(pages, rest, 32, 64), fp4.load(before, rest, 32, 64))


def with_4_bit_cache(monkeypatch):
    """The plain model attends over keys and values as a 4-bit cache holds them."""
    plain = plain_llama.causal_attention
    hold = lambda t: fp4_plain.quantized(t).to(t.dtype)  # noqa: E731
    monkeypatch.setattr(plain_llama, "causal_attention", lambda q, k, v: plain(q, hold(k), hold(v)))


@pytest.mark.parametrize("name", ["A", "B"])
def test_engine_with_a_4_bit_cache_is_the_plain_model_with_one(tmp_path, monkeypatch, name):
    from torchllms_b200.engine.replay import Replayer
    cfg, seed, _page = TINY[name]
    folder = tiny_folder(tmp_path, name)
    rng = random.Random(seed)
    reqs = {f"r{i}": [rng.randrange(cfg["vocab_size"]) for _ in range(n)] for i, n in enumerate([1, 7, 33, 64, 50])}
    model = plain_llama.PlainModel(folder)
    full = {rid: model.logits(t).numpy() for rid, t in reqs.items()}
    with_4_bit_cache(monkeypatch)
    held = {rid: model.logits(t).numpy() for rid, t in reqs.items()}
    steps, places, peak = traces.mixed(reqs)
    rp = Replayer(folder, "float32", peak + 16 * len(reqs), page_size=16, device="cpu", ops=Fp4TorchOps(), kv_format="fp4")
    off = moved = 0.0
    for s in steps:
        got = rp.run_step(s)
        rp.engine.cache.check_invariants()
        if s["step"] in places:
            want = np.stack([held[rid][pos] for rid, pos in places[s["step"]]])
            off = max(off, float(np.abs(got - want).mean()))
            moved = max(moved, float(np.abs(want - np.stack([full[rid][pos] for rid, pos in places[s["step"]]])).mean()))
    # sums in another order flip a code here and there; a wrong scale, row or key moves logits as far as the 4 bits do
    assert off < 0.1 * moved, (off, moved)


def test_llm_takes_the_format_and_others_refuse_it(tmp_path):
    from torchllms_b200.inference import LLM
    from torchllms_b200.inference.chat import parse_args
    folder = tiny_folder(tmp_path, "A")
    llm = LLM(folder, precision="float32", max_len=64, max_bsz=2, device="cpu", ops=Fp4TorchOps(), kv_cache="fp4", kv_memory_gb=1e-3)
    per_token = 2 * 2 * 2 * (8 + 1)                       # layers, k and v, heads, a head of 16
    assert llm.engine.cache.groups[0].allocator.n_pages == -(-(int(1e-3 * 2 ** 30) // per_token) // 16)
    out = llm.generate(prompt_token_ids=[[1, 2, 3], [4]], max_new_tokens=4)
    assert [len(r.token_ids) for r in out] == [4, 4] and all(r.error is None for r in out)
    with pytest.raises(ValueError, match="kv_cache must be one of"):
        LLM(folder, precision="float32", device="cpu", ops=Fp4TorchOps(), kv_cache="int4")
    with pytest.raises(ValueError, match="pages of a multiple"):
        LLM(folder, precision="float32", device="cpu", ops=Fp4TorchOps(), kv_cache="fp4", page_size=8)
    assert parse_args(["--ckpt_paths", "x", "--kv_cache", "fp4"]).kv_cache == "fp4" and parse_args(["--ckpt_paths", "x"]).kv_cache == "full"


def test_architectures_without_the_format_say_so(tmp_path):
    from nagolix_cases import CASES, case_folder
    from torchllms_b200.engine.loading import load_model
    folder = case_folder(tmp_path, next(iter(CASES)))[2]
    with pytest.raises(ValueError, match="no cache of format 'fp4'"):
        load_model(folder, dtype="float32", device="cpu", ops=Fp4TorchOps(), kv_format="fp4")
