"""A shared expert beside routed ones, weights in 8 bits: its result meets the experts' before it is rounded."""

import pytest
import torch

import rakuvik_cases
from test_fp8_weights import Fp8TorchOps
from torchllms_b200.engine.loading import load_model
from torchllms_b200.engine.replay import Replayer
from torchllms_b200.engine.step import StepEntry


class Watching(Fp8TorchOps):
    def moe_experts_fp8(self, x, chosen, weights, w_up, w_down, *, shared=None, **kw):
        self.shared = shared
        return super().moe_experts_fp8(x, chosen, weights, w_up, w_down, shared=shared, **kw)


def folder_of(tmp_path):
    cfg = rakuvik_cases.config([rakuvik_cases.attention_layer(mlp=rakuvik_cases.moe(ff=32, shared=48))], width=64)
    return rakuvik_cases.write_folder(tmp_path, "moe", cfg, rakuvik_cases.tensors_for(cfg, 1), torch.bfloat16)


def test_its_result_stays_in_32_bits(tmp_path):
    ops = Watching()
    _arch, _cfg, model = load_model(folder_of(tmp_path), dtype="bfloat16", device="cpu", ops=ops, weight_format="fp8")
    experts = next(p for b in model.blocks for p in b.parts_within() if type(p).__name__ == "RoutedExperts")
    x = torch.randn((5, 64), generator=torch.Generator().manual_seed(1)).bfloat16()
    out = experts.forward(x, None)
    assert ops.shared.dtype == torch.float32 and out.dtype == torch.bfloat16
    u = ops.linear_activation_fp8(x, experts.w_shared_up, experts.activation, gated=experts.gated, act_params=experts.shared_act_params)
    assert torch.equal(ops.shared, ops.linear_fp8(u, experts.w_shared_down, torch.float32))


@pytest.mark.gpu
def test_a_step_with_the_kernels(tmp_path):
    engine = Replayer(folder_of(tmp_path), "bfloat16", 512, weight_format="fp8").engine
    a = engine.claim()
    rows = engine.step([StepEntry(a, [(5 * i) % 97 for i in range(70)], [69])]).float().clone()
    engine.model.ops.check_status()
    assert bool(torch.isfinite(rows).all())
