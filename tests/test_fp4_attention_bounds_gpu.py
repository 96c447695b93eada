"""Attention over the 4-bit cache at its bounds: what a row does not see takes no part in it, whatever it is."""

import pytest
import torch

import fp4_plain
from test_fp4_kernels_gpu import batch, judge, ops
from torchllms_b200.cache import fp4

pytestmark = pytest.mark.gpu


def attend(a, kw, impl):
    """One call; ``impl`` may name a number of pieces."""
    pieces = dict(allow_split=int(impl.split()[2])) if "pieces" in impl else {}
    out = ops().paged_attention_fp4(**a, **kw, impl=impl.split()[0], **pieces)
    ops().check_status()
    return out


def poisoned(a, kw, share, seed):
    """The step with ``share`` of the value groups that requests hold made NaN, and where a result has to be NaN for it: in the
    coordinates of a group that is one at a key which the row sees."""
    g = torch.Generator().manual_seed(seed)
    T, H, D = a["q"].shape
    KV, page, window = a["k_pages"].shape[1], kw["page_size"], kw["window"]
    v_pages, wanted = a["v_pages"].clone(), torch.zeros((T, H, D), dtype=torch.bool)
    scales = fp4.rows_of(v_pages, D)[1]
    q_start, table = a["q_start"].tolist(), a["block_table"].cpu()
    for b, L in enumerate(a["kv_len"].tolist()):
        n = q_start[b + 1] - q_start[b]
        if L == 0 or n == 0:
            continue
        bad = torch.rand((L, KV, D // 16), generator=g) < share
        bad[L - 1, 0, 0] = bad[max(0, L - n), KV - 1, D // 16 - 1] = True          # (the last token, and the first new one)
        if window:
            bad[:max(0, L - n - window + 1)] = False                               # (no page holds those)
        for j, h, c in bad.nonzero().tolist():
            scales[int(table[b, j // page]), h, j % page // 16, j % 16, c] = fp4.NAN_SCALE
        for i in range(n):
            pos = L - n + i
            seen = bad[max(0, pos - window + 1) if window else 0:max(pos + 1, 0)].any(0)
            wanted[q_start[b] + i] = seen.repeat_interleave(16, 1).repeat_interleave(H // KV, 0)
    return dict(a, v_pages=v_pages), wanted


@pytest.mark.parametrize("share", [0.0, 0.002, 0.03])
@pytest.mark.parametrize("impl,dtype", [("general", "bf16"), ("general", "f32"), ("decode", "bf16"), ("decode", "f32"), ("prefill", "bf16"),
                                        ("prefill in 3 pieces", "bf16"), ("prefill in 7 pieces", "bf16"), ("auto", "bf16"), ("auto", "f32")])
@pytest.mark.parametrize("H,KV,D,page,q_lens,kv_lens,window", [
    pytest.param(2, 2, 64, 16, [300], [420], None, id="a_token_a_row"),
    pytest.param(9, 3, 128, 32, [40, 3, 1], [40, 200, 30], None, id="group_of_3"),
    pytest.param(32, 4, 64, 16, [130, 17], [130, 460], None, id="group_of_8"),
    pytest.param(12, 1, 128, 64, [4, 1, 2], [900, 333, 20], None, id="drafts"),
    pytest.param(8, 2, 128, 16, [90, 5], [700, 300], 100, id="window_100"),
    pytest.param(4, 4, 64, 16, [290], [800], 33, id="window_33"),
    pytest.param(6, 2, 128, 48, [64, 64], [64, 129], 1, id="window_1"),
    pytest.param(2, 2, 128, 16, [257], [600], 300, id="window_300"),
    pytest.param(4, 2, 64, 16, [5, 9, 3], [2, 70, 3], None, id="rows_that_see_nothing"),
    pytest.param(4, 2, 64, 16, [9, 70], [5, 30], 7, id="rows_that_see_nothing_in_a_window"),
    pytest.param(32, 8, 64, 16, [65, 0, 200, 7], [65, 30, 777, 7], None, id="prompts"),
])
def test_values_that_are_no_numbers_reach_the_rows_that_see_them_only(H, KV, D, page, q_lens, kv_lens, window, impl, dtype, share):
    a, kw = batch(H, KV, D, page, q_lens, kv_lens, window, dtype, seed=len(q_lens) + D)
    before = attend(a, kw, impl)
    b, wanted = poisoned(a, kw, share, seed=H + D)
    got = attend(b, kw, impl)
    assert torch.equal(got.isnan().cpu(), wanted)
    # everything else keeps its bits
    assert torch.equal(got[~wanted.cuda()], before[~wanted.cuda()])


@pytest.mark.parametrize("impl,dtype", [("general", "bf16"), ("decode", "bf16"), ("decode", "f32"), ("prefill", "bf16"), ("prefill in 3 pieces", "bf16")])
def test_a_window_of_any_size(impl, dtype):
    """A window that holds every key is no window, up to the largest number there is."""
    a, kw = batch(4, 2, 64, 16, [9, 70, 1], [5, 30, 90], None, dtype)
    whole = attend(a, kw, impl)
    for window in (90, 2 ** 20, 2 ** 31 - 1):
        assert torch.equal(attend(a, dict(kw, window=window), impl), whole)


@pytest.mark.parametrize("impl,dtype", [("general", "bf16"), ("decode", "bf16"), ("decode", "f32")])
@pytest.mark.parametrize("H,KV,D,most", [(4, 2, 64, 1), (7, 1, 128, 1), (7, 1, 64, 2), (3, 3, 128, 3)])
def test_requests_with_more_tokens_than_the_step_says(H, KV, D, most, impl, dtype):
    """Of a request that brings more than ``max_q_len`` tokens the first ones are computed, and nothing else is touched."""
    a, kw = batch(H, KV, D, 16, [3, 1, 9, 2], [300, 20, 90, 2], None, dtype)
    kw["max_q_len"] = most
    out = torch.full_like(a["q"], 9.0)
    got = ops().paged_attention_fp4(**a, **kw, impl=impl, out=out).double().cpu()
    ops().check_status()
    want, s, v = fp4_plain.attention(a["q"], a["k_pages"], a["v_pages"], a["block_table"], a["q_start"], a["kv_len"], 16, kw["scale"], None)
    bound = v * (s + 4.0) * 2.0 ** -18 + (v * 2.0 ** -12 + want.abs() * 2.0 ** -8 if dtype == "bf16" else 0.0)
    starts = a["q_start"].tolist()
    computed = torch.tensor([t - lo < most for lo, hi in zip(starts, starts[1:]) for t in range(lo, hi)])
    assert ((got - want).abs() <= bound)[computed].all() and (got[~computed] == 9.0).all()


@pytest.mark.parametrize("impl,dtype", [("general", "f32"), ("decode", "bf16"), ("decode", "f32"), ("prefill", "bf16"), ("prefill in 3 pieces", "bf16")])
@pytest.mark.parametrize("scale", [-0.125, 0.0, 1e-30, -1e-30])
def test_scales_that_are_not_positive(impl, dtype, scale):
    """The formula holds for any factor: negative ones, none at all, and ones that vanish beside small queries."""
    for sharp in (1.0, 1e-30, 0.0):
        a, kw = batch(8, 2, 64, 16, [1, 70, 3], [200, 150, 2], None, dtype, sharp=sharp)
        kw["scale"] = scale
        judge(attend(a, kw, impl), a, kw)


def test_scales_that_are_no_numbers_are_refused():
    from torchllms_b200.kernels.native import KernelError
    a, kw = batch(4, 2, 64, 16, [1], [30])
    for scale in (float("nan"), float("inf"), -float("inf"), 1e300):
        with pytest.raises(KernelError, match="finite float32"):
            ops().paged_attention_fp4(**a, **dict(kw, scale=scale))


def test_every_instance_has_its_own_status_word():
    """A call's bounded waits report to the instance that made the call, whichever instance made its first call last."""
    import ctypes
    from torchllms_b200.kernels.native import NativeOps
    seen = []
    signature = ctypes.CFUNCTYPE(ctypes.c_int, *[ctypes.c_void_p] * 4, ctypes.c_void_p, ctypes.c_int, ctypes.c_int, *[ctypes.c_void_p] * 5,
                                 *[ctypes.c_int] * 6, ctypes.c_longlong, ctypes.c_int, ctypes.c_int, ctypes.c_int, ctypes.c_float, ctypes.c_void_p)
    fake = signature(lambda *args: seen.append(args[11]) or 0)           # (the status word is the twelfth; nothing is launched)

    class Library:
        def __init__(self, real):
            self.real = real

        def __getattr__(self, name):
            return fake if name == "tl_attention_fp4_decode" else getattr(self.real, name)

    one, two = NativeOps(), NativeOps()
    for o in (one, two):
        load = o._lib
        o._lib = lambda name, load=load: Library(load(name)) if name == "attention_fp4_decode" else load(name)
    a, kw = batch(4, 2, 64, 16, [1], [30])
    try:
        for o in (one, two, one):
            o.paged_attention_fp4(**a, **kw, impl="decode")
    finally:
        ops()._fp4_load()                                                # (the kernels themselves again)
    assert seen == [o._status.data_ptr() for o in (one, two, one)]
    judge(ops().paged_attention_fp4(**a, **kw, impl="decode"), a, kw)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("n,behind", [(4, 3000), (16, 2500), (64, 1900), (200, 700)])
def test_a_portion_that_is_cut_leaves_the_rows_beside_it_alone(D, n, behind):
    """Decoded tokens and a portion in one output: the portion's keys are cut and its pieces added up over its own rows."""
    H, KV, page, nd = 8, 2, 16, 3
    a, kw = batch(H, KV, D, page, [1] * nd + [n], [40, 700, 1300, behind + n], None, "bf16", seed=n)
    part = lambda lo, hi: dict(a, block_table=a["block_table"][lo:hi], q_start=a["q_start"][lo:hi + 1], kv_len=a["kv_len"][lo:hi])  # noqa: E731
    out = torch.full_like(a["q"], 9.0)
    ops().paged_attention_fp4(**part(0, nd), **dict(kw, n_seqs=nd, max_q_len=1), n_tokens=nd, out=out)
    decoded = out[:nd].clone()
    for cut in (True, 5):
        before = ops().launches
        ops().paged_attention_fp4(**part(nd, nd + 1), **dict(kw, n_seqs=1), out=out, allow_split=cut, impl="prefill")
        assert ops().launches - before == 2 and torch.equal(out[:nd], decoded)
        judge(out, a, kw)
        out[nd:] = 9.0
    ops().paged_attention_fp4(**part(nd, nd + 1), **dict(kw, n_seqs=1), out=out)
    ops().check_status()
    assert torch.equal(out[:nd], decoded)
    judge(out, a, kw)


def test_keys_that_may_not_be_cut_go_to_the_kernel_that_is_faster_so():
    """(64 rows behind 12,000 keys: 8 CTAs of the tcgen05 kernel would walk all of them)"""
    a, kw = batch(8, 2, 64, 16, [16], [3000], None, "bf16")
    whole = ops().paged_attention_fp4(**a, **kw, allow_split=False)
    assert torch.equal(whole, ops().paged_attention_fp4(**a, **kw, impl="decode"))
    assert not torch.equal(whole, ops().paged_attention_fp4(**a, **kw, allow_split=False, impl="prefill"))
    a, kw = batch(8, 8, 64, 16, [300] * 4, [400] * 4, None, "bf16")                      # 300 rows of 32 units
    assert torch.equal(ops().paged_attention_fp4(**a, **kw, allow_split=False), ops().paged_attention_fp4(**a, **kw, allow_split=False, impl="prefill"))


@pytest.mark.parametrize("D,n,most_kv,kernel", [(128, 8, 200, "decode"), (128, 8, 1024, "decode"), (128, 8, 1025, "prefill"), (128, 8, 4096, "prefill"),
                                                (128, 15, 1024, "decode"), (128, 4, 4096, "decode"), (128, 16, 1024, "prefill"), (64, 15, 4096, "decode"),
                                                (64, 16, 1024, "prefill")])
def test_the_kernel_goes_by_rows_and_the_planned_context(D, n, most_kv, kernel):
    """(groups of four; a step may plan for more keys than its requests have)"""
    a, kw = batch(8, 2, D, 16, [n, n], [200, 150], None, "bf16", seed=n)
    a["block_table"] = torch.nn.functional.pad(a["block_table"], (0, 256), value=-1)
    kw["max_kv_len"] = most_kv
    got = {impl: ops().paged_attention_fp4(**a, **kw, impl=impl) for impl in ("auto", "decode", "prefill")}
    ops().check_status()
    judge(got["auto"], a, kw)
    assert not torch.equal(got["decode"], got["prefill"]) and torch.equal(got["auto"], got[kernel])


@pytest.mark.parametrize("impl,dtype", [("general", "bf16"), ("general", "f32"), ("decode", "bf16"), ("decode", "f32"), ("prefill", "bf16"), ("prefill in 3 pieces", "bf16")])
@pytest.mark.parametrize("H,KV,q_lens,kv_lens,window", [(4, 2, [1, 1, 1], [1, 300, 17], None), (4, 2, [5, 70, 9], [2, 70, 400], None),
                                                       (4, 2, [20, 3], [20, 90], 1), (32, 8, [65, 1, 200], [65, 30, 220], None)])
@pytest.mark.parametrize("value", ["nan", "inf", "-inf"])
def test_queries_that_are_not_finite(impl, dtype, H, KV, q_lens, kv_lens, window, value):
    """They give what softmax gives (NaN, also where every score is -inf; a row without a key is zeros) and leave the other rows' bits alone."""
    a, kw = batch(H, KV, 64, 16, q_lens, kv_lens, window, dtype, seed=len(q_lens))
    before = attend(a, kw, impl)
    g = torch.Generator().manual_seed(7)
    T = a["q"].shape[0]
    hit = torch.rand((T, H), generator=g) < 0.4
    hit[0, 1] = hit[-1, 2] = True
    where = torch.randint(0, 64, (T, H, 1), generator=g)
    q = a["q"].cpu().scatter(2, where, torch.where(hit[..., None], float(value), a["q"].cpu().gather(2, where).float()).to(a["q"].dtype))
    got = attend(dict(a, q=q.cuda()), kw, impl)
    position = []
    for b, L in enumerate(kv_lens):
        position += list(range(L - q_lens[b], L))
    wanted = hit & (torch.tensor(position) >= 0)[:, None]
    assert torch.equal(got.isnan().cpu(), wanted[..., None].expand(-1, -1, 64))
    assert torch.equal(got[~wanted.cuda()], before[~wanted.cuda()])
