"""Steps over a 4-bit cache that bring portions: what their calls of the attention are told, and recorded steps beside others."""

import pytest
import torch

from helpers import TINY_C, make_tensors, tiny_folder, write_model_folder
from test_fp4_cache import Fp4TorchOps
from torchllms_b200.engine.replay import Replayer
from torchllms_b200.engine.step import StepEntry


class Recording(Fp4TorchOps):
    """The plain twins, with what each attention call was told."""

    def __init__(self):
        super().__init__()
        self.calls, self.bounds = [], []

    def paged_attention(self, q, *args, **kw):
        self.bounds.append(kw["max_kv_len"])
        self.calls.append(("full", kw["n_seqs"], kw["max_q_len"], kw.get("allow_split", True)))
        return super().paged_attention(q, *args, **kw)

    def paged_attention_fp4(self, q, *args, **kw):
        out = super().paged_attention_fp4(q, *args, **kw)
        self.calls[-1] = ("fp4",) + self.calls[-1][1:]
        return out


@pytest.mark.parametrize("kv_format,cut", [("full", False), ("fp4", True)])
def test_keys_of_portions_beside_decoded_tokens_may_be_cut(tmp_path, kv_format, cut):
    """Two calls fill one output.  The cache in the compute type has a merge pass over all of it, so its portions' keys stay whole;
    the 4-bit cache's goes over its own call's rows."""
    ops = Recording()
    rp = Replayer(tiny_folder(tmp_path, "A"), "float32", 256, page_size=16, device="cpu", ops=ops, kv_format=kv_format)
    engine = rp.engine
    a, b = engine.claim(), engine.claim()
    engine.step([StepEntry(a, [1, 2, 3])])
    ops.calls.clear()
    engine.step([StepEntry(a, [4]), StepEntry(b, [5, 6, 7, 8, 9])])
    assert set(ops.calls) == {(kv_format, 1, 1, True), (kv_format, 1, 5, cut)}


@pytest.mark.parametrize("kv_format,bounds", [("full", {30, 42, 60}), ("fp4", {128})])
def test_portions_over_a_4_bit_cache_plan_for_a_bound(tmp_path, kv_format, bounds):
    """Recorded steps are told apart by what their launches were planned for: with a cache whose keys are cut for long portions,
    too, that is a bound of the context, not the length that the first such step happened to have."""
    ops = Recording()
    engine = Replayer(tiny_folder(tmp_path, "A"), "float32", 128, page_size=16, device="cpu", ops=ops, kv_format=kv_format).engine
    a = engine.claim()
    for n in (30, 12, 18):
        ops.bounds.clear()
        engine.step([StepEntry(a, [1 + i for i in range(n)])])
        if n > 16:
            assert set(ops.bounds) <= bounds, ops.bounds


def test_portions_beside_many_requests_plan_for_their_own_bound(tmp_path):
    """Short portions of many requests plan for the longest context there may be; a long one plans for what there is."""
    folder = write_model_folder(tmp_path / "long", dict(TINY_C, max_position_embeddings=4096), make_tensors(TINY_C, 2), torch.float32)
    ops = Recording()
    engine = Replayer(folder, "float32", 4096, page_size=16, device="cpu", ops=ops, kv_format="fp4", max_num_seqs=20).engine
    handles = [engine.claim() for _ in range(17)]
    for n, bound in ((3, 4096), (20, 1024)):
        ops.bounds.clear()
        engine.step([StepEntry(h, [1]) for h in handles[:-1]] + [StepEntry(handles[-1], list(range(1, n + 1)))])
        # (the one-token rows' own call plans for all of them either way)
        assert sorted(set(ops.bounds)) == sorted({4096, bound})


@pytest.mark.gpu
def test_a_step_recorded_at_a_short_context_is_not_the_one_of_a_long_one(tmp_path):
    """Portions of 48 tokens, one behind the other: recorded steps give the bits and make the launches of eager ones all the way."""
    folder = write_model_folder(tmp_path / "long", dict(TINY_C, max_position_embeddings=8192), make_tensors(TINY_C, 2), torch.bfloat16)
    runs = []
    for graphs in (False, True):
        engine = Replayer(folder, "bfloat16", 8192, page_size=16, kv_format="fp4").engine
        engine.use_graphs = engine.use_graphs and graphs
        assert engine.use_graphs == graphs
        a, run = engine.claim(), []
        for step in range(100):
            before = engine.model.ops.launches
            logits = engine.step([StepEntry(a, [(7 * step + i) % 777 for i in range(48)])]).clone()
            run.append((logits, engine.model.ops.launches - before))
        assert (engine.graph_replays > 50) == graphs
        runs.append(run)
    for (eager, launches), (recorded, as_many) in zip(*runs):
        assert launches == as_many and torch.equal(eager, recorded)
