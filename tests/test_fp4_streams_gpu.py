"""Calls of the 4-bit cache's operators beside each other: streams, graphs, repetition, and the libraries' debug builds."""

import os
import subprocess
import sys
from pathlib import Path

import pytest
import torch

from test_fp4_kernels_gpu import DT, batch, judge, ops
from torchllms_b200.cache import fp4

pytestmark = pytest.mark.gpu


def cases():
    """Steps whose requests are cut into parts that are counted, and one with pieces that a second kernel adds up."""
    g = torch.Generator().manual_seed(5)
    lens = lambda n, most: torch.randint(1, most, (n,), generator=g).tolist()  # noqa: E731
    return [batch(16, 4, 128, 16, [1] * 24, lens(24, 700), seed=61), batch(8, 2, 64, 16, [2] * 20, [2 + n for n in lens(20, 900)], dtype="f32", seed=62),
            batch(8, 2, 64, 16, [20, 70], [1500, 900], seed=63)]


def test_streams_and_graphs_do_not_meet():
    """Calls on several streams, and graphs of one capture stream that are replayed on several, run beside each other; memory that a
    graph's pool hands out again is not zero, and a call before any replay finds its counters in order."""
    made = [(dict(a, **kw), ops().paged_attention_fp4(**a, **kw)) for a, kw in cases()]
    for (a, kw), (_args, want) in zip(cases(), made):
        judge(want, a, kw)
    torch.cuda.synchronize()
    filled = torch.cuda.CUDAGraph()
    with torch.cuda.graph(filled):
        used = torch.full((1 << 20,), -1, dtype=torch.int32, device="cuda")
    filled.replay()
    torch.cuda.synchronize()
    del used
    graphs, outs = [], [[torch.empty_like(want) for _ in range(16)] for _args, want in made]
    for (args, _want), into in zip(made, outs):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], pool=filled.pool() if len(graphs) == 1 else None):
            for o in into:
                ops().paged_attention_fp4(**args, out=o)
    for args, want in made:
        assert torch.equal(ops().paged_attention_fp4(**args), want)
    streams = [torch.cuda.Stream() for _ in made]
    for replayed in (True, False):
        for _ in range(10):
            for into in outs:
                for o in into:
                    o.fill_(float("nan"))
            torch.cuda.synchronize()
            if replayed:
                for s, graph in zip(streams, graphs):
                    with torch.cuda.stream(s):
                        graph.replay()
            else:
                for i in range(16):
                    for s, (args, _want), into in zip(streams, made, outs):
                        with torch.cuda.stream(s):
                            ops().paged_attention_fp4(**args, out=into[i])
            torch.cuda.synchronize()
            for (_args, want), into in zip(made, outs):
                assert all(torch.equal(o, want) for o in into)
    ops().check_status()


@pytest.mark.parametrize("impl", ["general", "decode", "prefill", "prefill in 3 pieces"])
@pytest.mark.parametrize("H,KV,D,q_lens,kv_lens,window", [(8, 2, 128, [1] * 4, [3000, 900, 1, 2222], None), (8, 2, 64, [300, 65, 5], [900, 65, 700], None),
                                                         (4, 4, 128, [200], [1500], 333)])
def test_the_same_call_gives_the_same_bits(H, KV, D, q_lens, kv_lens, window, impl):
    """Whoever is last to finish a part, or first to need a new maximum."""
    a, kw = batch(H, KV, D, 16, q_lens, kv_lens, window)
    kw.update(impl=impl.split()[0], **(dict(allow_split=3) if "pieces" in impl else {}))
    first = ops().paged_attention_fp4(**a, **kw)
    for _ in range(20):
        assert torch.equal(ops().paged_attention_fp4(**a, **kw), first)
    ops().check_status()


@pytest.mark.parametrize("T,H,KV,D", [(1, 4, 2, 64), (17, 32, 8, 128), (200, 16, 4, 64), (600, 8, 8, 128)])
def test_what_is_written_is_what_the_next_calls_read(T, H, KV, D):
    """The same slots written again and again, each time read back and attended over at once, by kernels that start while the one
    before them still runs; eagerly and recorded."""
    page = 16
    g = torch.Generator(device="cuda").manual_seed(T)
    rows = [torch.randn((T, (H + 2 * KV) * D), generator=g, device="cuda").to(torch.bfloat16) for _ in range(8)]
    pages = [torch.zeros(fp4.page_shape(-(-T // page), KV, page, D), dtype=torch.uint8, device="cuda") for _ in range(2)]
    table, places = torch.randn((T, D // 2, 2), generator=g, device="cuda"), torch.arange(T, dtype=torch.int32, device="cuda")
    a = dict(block_table=torch.arange(pages[0].shape[0], dtype=torch.int32, device="cuda")[None], q_start=torch.tensor([0, T], dtype=torch.int32).cuda(),
             kv_len=torch.tensor([T], dtype=torch.int32).cuda(), n_seqs=1, max_q_len=T, max_kv_len=T, scale=D ** -0.5, window=None, page_size=page)

    def step(x):
        q = ops().rope_kv_write_fp4(x, places, table, n_heads=H, n_kv_heads=KV, head_dim=D, interleaved=True, k_pages=pages[0], v_pages=pages[1],
                                    slot_mapping=places, page_size=page)
        return [*ops().kv_read_fp4(pages[0], pages[1], places, head_dim=D, page_size=page, out_dtype=torch.bfloat16),
                *(ops().paged_attention_fp4(q, pages[0], pages[1], **a, impl=impl) for impl in ("general", "decode", "prefill"))]

    want = []
    for x in rows:
        torch.cuda.synchronize()
        want.append(step(x))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        recorded = [step(x) for x in rows]
    for _ in range(10):
        graph.replay()
        torch.cuda.synchronize()
        for got in ([step(x) for x in rows], recorded):
            torch.cuda.synchronize()
            assert all(torch.equal(x, y) for some, all_of in zip(got, want) for x, y in zip(some, all_of))
    ops().check_status()


def everything():
    """One call of each kernel of the operators, on sound input: what they give."""
    given = []
    for T, D, dtype, interleaved in ((3, 64, "bf16", True), (200, 128, "bf16", False), (160, 64, "f32", True), (5, 48, "f32", False)):
        H, KV, page = 4, 2, 32
        g = torch.Generator().manual_seed(T)
        x = torch.randn((T, (H + 2 * KV) * D), generator=g).to(DT[dtype]).cuda()
        table, positions = torch.randn((50, D // 2, 2), generator=g).cuda(), torch.randint(0, 50, (T,), generator=g).int().cuda()
        slots = torch.randperm(256, generator=g)[:T].int().cuda()
        pages = [torch.zeros(fp4.page_shape(8, KV, page, D), dtype=torch.uint8, device="cuda") for _ in range(2)]
        given.append(ops().rope_kv_write_fp4(x, positions, table, n_heads=H, n_kv_heads=KV, head_dim=D, interleaved=interleaved, k_pages=pages[0],
                                             v_pages=pages[1], slot_mapping=slots, page_size=page))
        given += [*pages, *ops().kv_read_fp4(pages[0], pages[1], slots, head_dim=D, page_size=page, out_dtype=DT[dtype])]
    for D, impl, dtype, q_lens, kv_lens, window in ((96, "auto", "f32", [3, 40], [70, 40], None), (64, "decode", "bf16", [1, 1], [500, 3], None),
                                                    (128, "decode", "f32", [2, 70], [400, 90], 64), (128, "prefill", "bf16", [130, 9], [300, 9], 100),
                                                    (64, "prefill", "bf16", [40], [2000], None)):
        a, kw = batch(8, 2, D, 16, q_lens, kv_lens, window, dtype)
        given.append(ops().paged_attention_fp4(**a, **kw, impl=impl))
    ops().check_status()
    return [t.cpu() for t in given]


def test_debug_builds_give_the_same_and_report_nothing(tmp_path):
    """Libraries with every index checked on the device: sound input only, as everywhere."""
    here = Path(__file__).resolve().parent
    code = ("import sys, torch; sys.path.insert(0, sys.argv[1]); import test_fp4_streams_gpu as t;"
            "assert t.ops().debug; torch.save(t.everything(), sys.argv[2]); from torchllms_b200.kernels.build import loaded_libraries;"
            "assert {'kv_fp4', 'attention_fp4', 'attention_fp4_decode', 'attention_fp4_prefill'} <= set(loaded_libraries())")
    out = subprocess.run([sys.executable, "-c", code, str(here), str(tmp_path / "debug.pt")], capture_output=True, text=True, timeout=1800,
                         cwd=here.parent, env=dict(os.environ, TORCHLLMS_B200_DEBUG="1", PYTHONPATH=str(here.parent)))
    assert out.returncode == 0, out.stderr[-3000:]
    checked = torch.load(tmp_path / "debug.pt")
    release = everything()
    assert len(checked) == len(release) and all(torch.equal(x, y) for x, y in zip(checked, release))
