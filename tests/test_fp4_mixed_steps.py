"""Steps that have decoded tokens beside portions, over a 4-bit cache: which calls of the attention they make (on the host)."""

import pytest

from helpers import tiny_folder
from test_fp4_cache import Fp4TorchOps
from torchllms_b200.engine.replay import Replayer


class Recording(Fp4TorchOps):
    """The plain twins, with what each attention call was told."""

    def __init__(self):
        super().__init__()
        self.calls = []

    def paged_attention(self, q, *args, **kw):
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
    from torchllms_b200.engine.step import StepEntry
    a, b = engine.claim(), engine.claim()
    engine.step([StepEntry(a, [1, 2, 3])])
    ops.calls.clear()
    engine.step([StepEntry(a, [4]), StepEntry(b, [5, 6, 7, 8, 9])])
    assert set(ops.calls) == {(kv_format, 1, 1, True), (kv_format, 1, 5, cut)}
