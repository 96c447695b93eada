"""Calls of the 8-bit rows' operators beside each other: what is refused, streams, graphs, repetition, large offsets, a run of them together."""

import pytest
import torch

import fp8_plain as plain
from torchllms_b200.kernels.native import KernelError
from torchllms_b200.weights.fp8 import SCALES, Fp8Rows, encode

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from torchllms_b200.kernels import get_ops
    return get_ops()


def rand(shape, dtype=torch.float32, seed=0, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)


def held(x):
    return Fp8Rows(*encode(x))


def test_refusals(ops):
    x, w = rand((4, 256)), held(rand((32, 256), seed=1))
    rows = held(x)
    before = ops.launches
    flat = rand((4 * 256 + 4,))
    moved = flat[4:].view(4, 256)                                         # (16 bytes in, fine)
    bad = [
        (lambda: ops.quantize_fp8(x[:, ::2]), "contiguous"), (lambda: ops.quantize_fp8(x.half()), "float32/bfloat16"),
        (lambda: ops.quantize_fp8(rand((4, 120))), "multiple of 16"), (lambda: ops.quantize_fp8(x[0]), "matrix"),
        (lambda: ops.quantize_fp8(flat[1:1 + 4 * 256].view(4, 256)), "16 bytes"), (lambda: ops.quantize_fp8(x.cpu()), "GPU"),
        (lambda: ops.activation_fp8(rand((4, 48)), "silu", gated=True), "multiple of 16"), (lambda: ops.activation_fp8(x, "swish"), "unknown activation"),
        (lambda: ops.activation_fp8(x, "clamped_swish"), "clamped"), (lambda: ops.activation_fp8(x, "clamped_swish", gated=True, act_params=(0.0, 1.0, 0.0)), "clamped"),
        (lambda: ops.rmsnorm_fp8(x.bfloat16(), None, x[0], 1e-5), "float32"), (lambda: ops.rmsnorm_fp8(x, None, rand((128,)), 1e-5), "weight"),
        (lambda: ops.rmsnorm_fp8(x, rand((4, 128)), x[0], 1e-5), "delta"), (lambda: ops.rmsnorm_fp8(x, rand((2, 4, 256), torch.bfloat16), x[0], 1e-5), "partial sums"),
        (lambda: ops.rmsnorm_fp8(rand((1, 32784)), None, rand((32784,)), 1e-5), "registers"), (lambda: ops.rmsnorm_fp8(x, None, x[0], "a"), "eps"),
        (lambda: ops.linear_fp8(rows, w, out_dtype=torch.float16), "output dtype"), (lambda: ops.linear_fp8(rows, w, impl="best"), "impl"),
        (lambda: ops.linear_fp8(rows, rows.dequantize()), "8-bit rows"), (lambda: ops.linear_fp8(held(rand((4, 128))), w), "inner sizes"),
        (lambda: ops.linear_fp8(Fp8Rows(rows.codes, rows.scales[:, :2]), w), "contiguous"),
        (lambda: ops.linear_fp8(Fp8Rows(rows.codes, rows.scales[:2]), w), "scales"),
        (lambda: ops.linear_fp8(Fp8Rows(rows.codes, rows.scales.view(torch.uint8)), w), "float8_e8m0fnu"),
        (lambda: ops.linear_fp8(Fp8Rows(rows.codes.cpu(), rows.scales.cpu()), w), "GPU"),
        (lambda: ops.linear_activation_fp8(rows, held(rand((40, 256))), "silu"), "multiple of 16"),
        (lambda: ops.linear_activation_fp8(rows, held(rand((48, 256))), "silu", gated=True), "multiple of 16"),
        (lambda: ops.linear_activation_fp8(rows, w, "silu", impl="split"), "unsupported size"),
    ]
    up, down = held(rand((3, 32, 256))), held(rand((3, 256, 32)))
    chosen, share = torch.zeros((4, 2), dtype=torch.int32, device="cuda"), torch.ones((4, 2), device="cuda")
    call = lambda **kw: ops.moe_experts_fp8(**{**dict(x=x, chosen=chosen, weights=share, w_up=up, w_down=down, activation="silu"), **kw})  # noqa: E731
    assert call().shape == (4, 256)
    bad += [(lambda: call(chosen=chosen.long()), "int32"), (lambda: call(weights=share[:, :1]), "contiguous"), (lambda: call(chosen=chosen[:3]), "chosen and weights"),
            (lambda: call(w_down=up), "w_up"), (lambda: call(gated=True), "w_up"), (lambda: call(impl="split"), "unsupported size"),
            (lambda: call(shared=rand((4, 128))), "shared"), (lambda: call(shared_gate=torch.ones(4, device="cuda")), "shared expert"),
            (lambda: call(activation="clamped_swish"), "clamped"), (lambda: call(w_up=rand((3, 32, 256))), "8-bit rows")]
    launched = ops.launches
    for k, (f, what) in enumerate(bad):
        with pytest.raises(KernelError, match=what):
            f()
            pytest.fail(f"case {k} ({what}) was not refused")
    assert ops.launches == launched and launched == before + 5
    assert torch.equal(ops.quantize_fp8(moved).codes.view(torch.uint8), encode(moved)[0].view(torch.uint8))


def test_nothing_to_do(ops):
    w = held(rand((32, 256)))
    empty = torch.empty((0, 256), device="cuda")
    assert ops.linear_fp8(empty, w).shape == (0, 32) and ops.linear_fp8(held(empty), w, torch.float32).dtype == torch.float32
    assert ops.linear_activation_fp8(empty, w, "silu", gated=True).shape == (0, 16)
    assert ops.rmsnorm_fp8(empty, None, torch.ones(256, device="cuda"), 1e-5).scales.shape == (0, 4)
    assert ops.linear_fp8(held(rand((3, 256))), w[0:0]).shape == (3, 0)


def chain(ops, s):
    """A layer's feed-forward and a routed one, as they are used together."""
    rows = ops.rmsnorm_fp8(s["h"], s["delta"], s["norm"], 1e-5)
    y = ops.linear_fp8(ops.linear_activation_fp8(rows, s["w13"], "silu", gated=True), s["w2"])
    z = ops.moe_experts_fp8(y, s["chosen"], s["share"], s["up"], s["down"], activation="relu2")
    return ops.rmsnorm_fp8(s["h"], z, s["norm"], 1e-5), y, z


def material(T, seed=0, dim=512, hidden=640, E=8):
    score = rand((T, E), seed=seed + 9)
    best, chosen = torch.topk(score, 2, dim=-1)
    return dict(h=rand((T, dim), seed=seed), delta=rand((T, dim), torch.bfloat16, seed=seed + 1), norm=1.0 + 0.1 * rand((dim,), seed=3),
                w13=held(rand((2 * hidden, dim), seed=4, scale=dim ** -0.5)), w2=held(rand((dim, hidden), seed=5, scale=hidden ** -0.5)),
                up=held(rand((E, hidden, dim), seed=6, scale=dim ** -0.5)), down=held(rand((E, dim, hidden), seed=7, scale=hidden ** -0.5)),
                chosen=chosen.int().contiguous(), share=torch.softmax(best, -1).contiguous())


@pytest.mark.parametrize("T", [1, 5, 70, 300])
def test_a_run_of_them_together(ops, T):
    """Each operator's result against the definition on what the one before it left."""
    s = material(T)
    h0 = s["h"].double() + s["delta"].double()
    rows, y, z = chain(ops, s)
    ops.check_status()
    assert bool(((s["h"].double() - (h0 + z.double())).abs() <= 2.0 ** -22 * (h0.abs() + z.double().abs() + s["delta"].double().abs())).all())
    first = ops.rmsnorm_fp8(h0.float(), None, s["norm"], 1e-5)
    want, dy = plain.activated(plain.value(first), plain.value(s["w13"]), "silu", True)
    off = plain.moved(want, dy)
    w2 = plain.value(s["w2"])
    want_y, size = plain.stands_for(want) @ w2.T, (want.abs() + off) @ w2.abs().T
    assert bool(((y.double() - want_y).abs() <= off @ w2.abs().T + size * 24 * 2.0 ** -24 + want_y.abs() * 2.0 ** -8 * 1.01).all())
    want_z = plain.experts(y, s["chosen"], s["share"], plain.value(s["up"]), plain.value(s["down"]), "relu2")
    bound = plain.experts_bound(y, s["chosen"], s["share"], plain.value(s["up"]), plain.value(s["down"]), "relu2", result_eps=2.0 ** -8 * 1.01)
    assert bool(((z.double() - want_z).abs() <= bound).all())


def test_repetition_gives_the_same_bits(ops):
    runs = []
    for _ in range(20):
        s = material(37)
        rows, y, z = chain(ops, s)
        runs.append((rows.codes.view(torch.uint8), rows.scales.view(torch.uint8), y, z, s["h"]))
    ops.check_status()
    assert all(torch.equal(a, b) for run in runs[1:] for a, b in zip(run, runs[0]))


@pytest.mark.parametrize("T", [3, 200])
def test_a_recorded_run_is_the_eager_one(ops, T):
    s = material(T)
    start, delta = s["h"].clone(), s["delta"].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        chain(ops, s)
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):                                     # (two captures of the same calls, replayed in turn)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = chain(ops, s)
        graphs.append((g, out))
    for seed in (0, 20, 40):
        fresh = material(T, seed)
        s["delta"].copy_(fresh["delta"])
        s["chosen"].copy_(fresh["chosen"])
        for g, (rows, y, z) in graphs + graphs[:1]:
            s["h"].copy_(fresh["h"])
            g.replay()
            want = dict(s, h=fresh["h"].clone())
            w_rows, w_y, w_z = chain(ops, want)
            assert torch.equal(y, w_y) and torch.equal(z, w_z) and torch.equal(s["h"], want["h"])
            assert torch.equal(rows.codes.view(torch.uint8), w_rows.codes.view(torch.uint8))
    ops.check_status()
    assert start.shape == delta.shape


def test_streams_beside_each_other(ops):
    mats = [material(T, seed=100 * T) for T in (2, 40, 260)]
    want = []
    for s in mats:
        h = s["h"].clone()
        want.append(chain(ops, dict(s, h=h))[1:] + (h,))
    streams = [torch.cuda.Stream() for _ in mats]
    torch.cuda.synchronize()
    got = [[] for _ in mats]
    for _ in range(8):
        for k, (s, stream) in enumerate(zip(mats, streams)):
            with torch.cuda.stream(stream):
                h = s["h"].clone()
                got[k].append(chain(ops, dict(s, h=h))[1:] + (h,))
    torch.cuda.synchronize()
    ops.check_status()
    for runs, w in zip(got, want):
        assert all(torch.equal(a, b) for run in runs for a, b in zip(run, w))


def test_parts_of_a_weight(ops):
    """Slices of rows are views: their scales start where they start."""
    x, w = held(rand((33, 1040), seed=1)), held(rand((700, 1040), seed=2))
    whole = ops.linear_fp8(x, w, torch.float32, impl="single")
    for a, b in ((0, 128), (1, 130), (333, 700)):
        assert torch.equal(ops.linear_fp8(x, w[a:b], torch.float32, impl="single"), whole[:, a:b])
    assert torch.equal(ops.linear_fp8(x[5:20], w, torch.float32, impl="single"), whole[5:20])


def test_offsets_beyond_32_bits(ops):
    """Rows behind the first 2^31 bytes of codes, and results behind 2^31 numbers."""
    rows, K = 70000, 32768
    x = torch.empty((rows, K), dtype=torch.bfloat16, device="cuda")
    x.copy_(rand((1, K), torch.bfloat16, seed=1))
    x[-300:] = rand((300, K), torch.bfloat16, seed=2)
    held_rows = ops.quantize_fp8(x)
    codes, scales = encode(x[-300:])
    assert torch.equal(held_rows.codes[-300:].view(torch.uint8), codes.view(torch.uint8)) and torch.equal(held_rows.scales[-300:].view(torch.uint8), scales.view(torch.uint8))
    del x
    w = held(rand((144, K), seed=3, scale=K ** -0.5))
    for impl in ("single", "pair"):
        out = ops.linear_fp8(held_rows, w, impl=impl)
        assert torch.equal(out[-300:], ops.linear_fp8(held_rows[rows - 300:], w, impl=impl))
    few = Fp8Rows(held_rows.codes[:, :256].contiguous(), held_rows.scales[:, :4].contiguous())
    del held_rows
    wide = held(rand((32000, 256), seed=4, scale=1 / 16))
    out = ops.linear_fp8(few, wide)
    assert out.numel() > 2 ** 31 and torch.equal(out[-300:], ops.linear_fp8(few[rows - 300:], wide, impl="pair"))
    ops.check_status()


def test_experts_that_there_are_not_stay_in_bounds(ops):
    """A number beyond the experts: the token's result is not defined, the others' are what they are."""
    s = material(20)
    want = ops.moe_experts_fp8(s["delta"], s["chosen"], s["share"], s["up"], s["down"], activation="relu2")
    odd = s["chosen"].clone()
    odd[7, 1], odd[11, 0] = 8, -3
    got = ops.moe_experts_fp8(s["delta"], odd, s["share"], s["up"], s["down"], activation="relu2")
    keep = torch.ones(20, dtype=torch.bool, device="cuda")
    keep[7] = keep[11] = False
    assert torch.equal(got[keep], want[keep])


def test_many_experts(ops):
    """More experts than one pass of counters holds, most of them with no token."""
    E, T = 3000, 50
    up, down = held(rand((E, 16, 32), seed=1)), held(rand((E, 32, 16), seed=2))
    chosen = torch.randint(0, E, (T, 3), generator=torch.Generator(device="cuda").manual_seed(3), device="cuda", dtype=torch.int32)
    share, x = torch.rand((T, 3), device="cuda"), rand((T, 32), seed=4)
    got = ops.moe_experts_fp8(x, chosen, share, up, down, activation="gelu")
    want = plain.experts(x, chosen, share, plain.value(up), plain.value(down), "gelu")
    bound = plain.experts_bound(x, chosen, share, plain.value(up), plain.value(down), "gelu", result_eps=2.0 ** -24)
    assert bool(((got.double() - want).abs() <= bound + 1e-30).all())
    assert up.scales.dtype == SCALES
