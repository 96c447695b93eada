"""Weights in 8 bits through the engine: the option's way from its user to the parts, what is refused, and the engine's logits."""

import pytest
import torch

import fp8_plain as plain
import bomotar_cases
import lagusun_cases
import nunosun_cases
import rakuvik_cases
import zusitar_cases
from helpers import TINY, TINY_C, make_tensors, tiny_folder, write_model_folder
from torch_ops import TorchOps
from torchllms_b200.engine.loading import load_model
from torchllms_b200.engine.replay import Replayer
from torchllms_b200.engine.step import StepEntry
from torchllms_b200.inference import LLM
from torchllms_b200.inference.chat import parse_args
from torchllms_b200.kernels.lazy import PendingProduct
from torchllms_b200.parts.attention import PagedAttention
from torchllms_b200.parts.pair import SideBySide
from torchllms_b200.weights.fp8 import Fp8Rows, encode


class Fp8TorchOps(TorchOps):
    """The plain twins with weights in 8 bits, and the names of what was called."""

    def __init__(self):
        super().__init__()
        self.called = []

    def prepare(self, dtype, sampling=True, kv_format="full", weight_format="full"):
        self.called.append(("prepare", weight_format))

    def quantize_fp8(self, x):
        return Fp8Rows(*encode(x))

    def rmsnorm_fp8(self, h, delta, weight, eps):
        self.called.append("rmsnorm_fp8")
        if isinstance(delta, PendingProduct):
            delta = delta.take(self)
        if delta is not None:
            h += delta.float().sum(0) if delta.dim() == 3 else delta.float()
        return self.quantize_fp8(h * torch.rsqrt((h * h).mean(-1, keepdim=True) + eps) * weight)

    def linear(self, x, w, out_dtype=None, partials_ok=False):
        return self.linear_fp8(x, w, out_dtype or torch.bfloat16) if isinstance(w, Fp8Rows) else super().linear(x, w, out_dtype, partials_ok)

    def linear_fp8(self, x, w, out_dtype=torch.bfloat16):
        self.called.append("linear_fp8")
        x = x if isinstance(x, Fp8Rows) else self.quantize_fp8(x)
        return (x.dequantize() @ w.dequantize().t()).to(out_dtype)

    def linear_activation_fp8(self, x, w, activation, *, gated=False, act_params=None):
        self.called.append("linear_activation_fp8")
        return self.quantize_fp8(plain.act(self.linear_fp8(x, w, torch.float32), activation, gated, act_params))

    def moe_experts_fp8(self, x, chosen, weights, w_up, w_down, *, activation, shared=None, shared_gate=None, gated=False, act_params=None):
        self.called.append("moe_experts_fp8")
        out = plain.experts(x, chosen, weights, plain.value(w_up), plain.value(w_down), activation, gated, act_params)
        if shared is not None:
            extra = shared.double().sum(0) if shared.dim() == 3 else shared.double()
            out = out + (extra if shared_gate is None else extra * shared_gate.double()[:, None])
        return out.to(x.dtype)


def held_folder(tmp, cfg, tensors):
    """The model with every matrix of its layers as 8 bits hold it."""
    out = {k: Fp8Rows(*encode(v.to(torch.bfloat16))).dequantize() if v.dim() == 2 and k.startswith("layers.") else v for k, v in tensors.items()}
    return write_model_folder(tmp, cfg, out, torch.bfloat16)


def logits_of(folder, prompts, ops=None, device="cpu", **kw):
    engine = Replayer(folder, "bfloat16", 512, device=device, ops=ops, **kw).engine
    handles = [engine.claim() for _ in prompts]
    rows = [engine.step([StepEntry(h, p, [len(p) - 1]) for h, p in zip(handles, prompts)]).float().clone()]
    for t in (5, 17):
        rows.append(engine.step([StepEntry(h, [t + i], [0]) for i, h in enumerate(handles)]).float().clone())
    return torch.stack(rows), engine


PROMPTS = [[5, 17, 3, 700, 0, 41], [(7 * i) % 777 for i in range(150)], [7]]


def apart(a, b):
    return float((a - b).norm() / b.norm())


def test_the_engine_holds_and_calls(tmp_path):
    cfg, tensors = TINY_C, make_tensors(TINY_C, 2)
    folder = write_model_folder(tmp_path / "plain", cfg, tensors, torch.bfloat16)
    ops = Fp8TorchOps()
    got, engine = logits_of(folder, PROMPTS, ops, weight_format="fp8")
    assert set(c for c in ops.called if isinstance(c, str)) == {"rmsnorm_fp8", "linear_fp8", "linear_activation_fp8"}
    full, plain_engine = logits_of(folder, PROMPTS, TorchOps())
    matrices = sum(v.numel() for k, v in tensors.items() if v.dim() == 2 and k.startswith("layers."))
    scales = engine.model.weight_bytes() - (plain_engine.model.weight_bytes() - 2 * matrices) - matrices
    rows = sum(v.shape[0] * plain.pitch(v.shape[1]) for k, v in tensors.items() if v.dim() == 2 and k.startswith("layers."))
    assert scales == rows
    # rows that meet a matrix are held to 2^-4 of a number (0.6 of that on average, over sqrt(3)): 2.2 % a product, and the weights' own
    # as much; four products behind one another in each of two layers: some 9 %
    assert apart(got, full) < 0.25
    assert apart(got, logits_of(held_folder(tmp_path / "held", cfg, tensors), PROMPTS, TorchOps())[0]) < 0.2


def test_routed_experts_are_held(tmp_path):
    cfg = rakuvik_cases.config([rakuvik_cases.attention_layer(mlp=rakuvik_cases.moe(ff=32, shared=48))], width=64)
    folder = rakuvik_cases.write_folder(tmp_path, "moe", cfg, rakuvik_cases.tensors_for(cfg, 1), torch.bfloat16)
    ops = Fp8TorchOps()
    _arch, _cfg, model = load_model(folder, dtype="bfloat16", device="cpu", ops=ops, weight_format="fp8")
    experts = [p for b in model.blocks for p in b.parts_within() if type(p).__name__ == "RoutedExperts"]
    assert experts and all(type(p.w_up) is Fp8Rows and type(p.w_down) is Fp8Rows and type(p.w_shared_up) is Fp8Rows for p in experts)
    got, _engine = logits_of(folder, [[5, 7, 11, 2, 3], [1]], ops, weight_format="fp8")
    assert "moe_experts_fp8" in ops.called
    full, _engine = logits_of(folder, [[5, 7, 11, 2, 3], [1]], TorchOps())
    assert apart(got, full) < 0.25


def test_the_options_way(tmp_path):
    folder = write_model_folder(tmp_path / "m", TINY_C, make_tensors(TINY_C, 2), torch.bfloat16)
    ops = Fp8TorchOps()
    llm = LLM(folder, precision="bfloat16", max_len=128, max_bsz=2, device="cpu", ops=ops, weights="fp8")
    assert llm.model.weight_format == "fp8" and ("prepare", "fp8") in ops.called
    assert parse_args(["--ckpt_paths", "x", "--weights", "fp8"]).weights == "fp8" and parse_args(["--ckpt_paths", "x"]).weights == "full"
    out = llm.generate(prompt_token_ids=[[1, 2, 3], [4]], max_new_tokens=3)
    assert all(len(r.token_ids) == 3 for r in out)


def test_what_is_refused(tmp_path):
    folder = write_model_folder(tmp_path / "m", TINY_C, make_tensors(TINY_C, 2), torch.bfloat16)
    with pytest.raises(ValueError, match="weights must be one of"):
        LLM(folder, device="cpu", ops=Fp8TorchOps(), weights="int8")
    with pytest.raises(ValueError, match="bfloat16"):
        LLM(folder, device="cpu", precision="float32", ops=Fp8TorchOps(), weights="fp8")
    with pytest.raises(ValueError, match="multiple of 16"):
        LLM(tiny_folder(tmp_path, "D"), device="cpu", ops=Fp8TorchOps(), weights="fp8")
    cfg = rakuvik_cases.config([rakuvik_cases.attention_layer(mlp=rakuvik_cases.dense())], width=64)
    dense = rakuvik_cases.write_folder(tmp_path, "dense", cfg, rakuvik_cases.tensors_for(cfg, 1), torch.bfloat16)
    with pytest.raises(ValueError, match="no part of this architecture"):
        LLM(dense, device="cpu", ops=Fp8TorchOps(), weights="fp8")


def test_a_part_inside_a_pair_is_found():
    """A model whose only matrices in 8 bits are those of one of two mixers side by side is not refused."""
    pair, members = object.__new__(SideBySide), [object.__new__(PagedAttention) for _ in range(2)]
    pair.members = (("left", members[0]), ("right", members[1]))
    assert list(pair.parts_within()) == [pair, *members]


def expert_family(tmp, name, width=48):
    """A folder of each family that has routed experts, their widths a multiple of 16."""
    if name == "rakuvik":
        c, layers = rakuvik_cases, [rakuvik_cases.attention_layer(mlp=rakuvik_cases.moe(ff=32, shared=48))]
    elif name == "nunosun":
        c, layers = nunosun_cases, [nunosun_cases.parallel_layer(mlp=nunosun_cases.moe(ff=32)), nunosun_cases.delta_layer(mlp=nunosun_cases.moe(ff=16))]
    elif name == "zusitar":
        c, layers = zusitar_cases, [zusitar_cases.attention_layer(mlp=zusitar_cases.moe(ff=32, shared=(16, 1.2))),
                                    zusitar_cases.scan_layer(mlp=zusitar_cases.moe(ff=16, shared=(32, 1.2)))]
    elif name == "lagusun":
        c, layers = lagusun_cases, [lagusun_cases.windowed(mlp=lagusun_cases.moe(ff=32, shared=16)), lagusun_cases.chunked(mlp=lagusun_cases.moe(ff=16, shared=32))]
    else:
        c, layers = bomotar_cases, [bomotar_cases.layer(mlp=bomotar_cases.moe(ff=32)), bomotar_cases.layer(mlp=bomotar_cases.moe(ff=16))]
    cfg = c.config(layers, width=width)
    return c.write_folder(tmp, name, cfg, c.tensors_for(cfg, 1), torch.bfloat16)


FAMILIES = ("rakuvik", "nunosun", "zusitar", "lagusun", "bomotar")


# ------------------------------------------------------------------------------------------------- on a GPU

@pytest.mark.gpu
def test_logits_of_the_kernels(tmp_path):
    """The kernels' engine against the twins' on the same held weights.  Both round rows to bfloat16 in places of their own, 2^-9 of a number,
    which moves one number in 30 to another of E4M3, 2^-3 of it: 1.5 % a product at most, some 4 % behind eight of them."""
    folder = write_model_folder(tmp_path / "m", TINY_C, make_tensors(TINY_C, 2), torch.bfloat16)
    got, engine = logits_of(folder, PROMPTS, device="cuda", weight_format="fp8")
    engine.model.ops.check_status()
    want, _engine = logits_of(folder, PROMPTS, Fp8TorchOps(), device="cuda", weight_format="fp8")
    assert apart(got, want) < 0.08
    assert apart(got, logits_of(held_folder(tmp_path / "held", TINY_C, make_tensors(TINY_C, 2)), PROMPTS, device="cuda")[0]) < 0.2


@pytest.mark.gpu
def test_logits_of_experts(tmp_path):
    cfg = rakuvik_cases.config([rakuvik_cases.attention_layer(mlp=rakuvik_cases.moe(ff=32, shared=48))], width=64)
    folder = rakuvik_cases.write_folder(tmp_path, "moe", cfg, rakuvik_cases.tensors_for(cfg, 1), torch.bfloat16)
    prompts = [[(5 * i) % 97 for i in range(100)], [1, 2]]
    got, engine = logits_of(folder, prompts, device="cuda", weight_format="fp8")
    engine.model.ops.check_status()
    assert apart(got, logits_of(folder, prompts, device="cuda")[0]) < 0.25


@pytest.mark.gpu
def test_recorded_steps_are_eager_ones(tmp_path):
    """Decode steps and portions replayed from graphs give the bits of eager ones."""
    folder = write_model_folder(tmp_path / "m", TINY_C, make_tensors(TINY_C, 2), torch.bfloat16)
    runs = []
    for graphs in (False, True):
        engine = Replayer(folder, "bfloat16", 1024, weight_format="fp8").engine
        engine.use_graphs = engine.use_graphs and graphs
        assert engine.use_graphs == graphs
        a, b, run = engine.claim(), engine.claim(), []
        for step in range(20):
            tokens = [(7 * step + i) % 777 for i in range(30 if step % 5 == 0 else 1)]
            run.append(engine.step([StepEntry(a, tokens, [len(tokens) - 1]), StepEntry(b, [step], [0])]).clone())
        engine.model.ops.check_status()
        runs.append((run, engine.graph_replays))
    assert runs[0][1] == 0 and runs[1][1] > 5
    assert all(torch.equal(x, y) for x, y in zip(runs[0][0], runs[1][0]))


@pytest.mark.gpu
def test_generation(tmp_path):
    """Requests in a batch, cut into portions, beside keys and values in 4 bits: all are answered and no wait ran out."""
    folder = write_model_folder(tmp_path / "m", TINY_C, make_tensors(TINY_C, 2, std=0.05, qk_std=0.25), torch.bfloat16)
    llm = LLM(folder, precision="bfloat16", max_len=256, max_bsz=4, max_num_batched_tokens=64, prefill_chunk=48, weights="fp8", kv_cache="fp4")
    llm.warmup(batch_sizes=[3])
    out = llm.generate(prompt_token_ids=PROMPTS, max_new_tokens=8)
    assert all(r.error is None and len(r.token_ids) == 8 for r in out)
    llm.engine.model.ops.check_status()


@pytest.mark.gpu
@pytest.mark.parametrize("name", FAMILIES)
def test_every_family_with_experts(tmp_path, name):
    """Its experts are held and run; recorded steps give the bits of eager ones, and every number is one."""
    folder, runs = expert_family(tmp_path, name), []
    for graphs in (False, True):
        engine = Replayer(folder, "bfloat16", 512, weight_format="fp8").engine
        engine.use_graphs = engine.use_graphs and graphs
        held = [p for b in engine.model.blocks for p in b.parts_within() if type(p).__name__ == "RoutedExperts"]
        assert held and all(type(p.w_up) is Fp8Rows for p in held)
        a, b = engine.claim(), engine.claim()
        run = [engine.step([StepEntry(a, [(5 * i) % 83 for i in range(70)], [69]), StepEntry(b, [1, 2], [1])]).clone()]
        run += [engine.step([StepEntry(a, [s], [0]), StepEntry(b, [s + 20], [0])]).clone() for s in range(6)]
        engine.model.ops.check_status()
        runs.append(torch.stack(run))
    assert bool(torch.isfinite(runs[0]).all()) and torch.equal(*runs)
