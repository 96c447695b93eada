"""The kernels around weights in 8 bits against their definitions in 64 bits (fp8_plain)."""

import math

import pytest
import torch

import fp8_plain as plain
from torchllms_b200.weights.fp8 import Fp8Rows, encode, scale_pitch

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16]


@pytest.fixture(scope="module")
def ops():
    from torchllms_b200.kernels import get_ops
    return get_ops()


def rand(shape, dtype=torch.float32, seed=0, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)


def uneven(T, K, dtype=torch.float32, seed=0):
    """Rows whose channels differ in size, as activations do."""
    return (rand((T, K), seed=seed) * torch.exp(1.5 * rand((K,), seed=seed + 1))).to(dtype)


def held(x):
    return Fp8Rows(*encode(x))


def same_rows(rows, x):
    """The rows hold 64-bit ``x`` exactly as the format says, down to the byte of every scale."""
    codes, e = plain.hold(x.double())
    assert rows.codes.shape == x.shape and rows.scales.shape == (x.shape[0], plain.pitch(x.shape[1]))
    want = torch.zeros(rows.scales.shape, dtype=torch.uint8, device=x.device)
    want[:, :e.shape[1]] = (e + 127).to(torch.uint8)
    assert torch.equal(rows.scales.view(torch.uint8), want)
    assert torch.equal(rows.codes.double().nan_to_num(777.0), codes.nan_to_num(777.0))


def near_rows(rows, y, slack):
    """The rows hold 64-bit ``y`` up to a relative error ``slack`` of what was rounded: half a step of E4M3 (2^-4 of the number, or
    2^-10 of the block's scale) and that much more."""
    got, scale = plain.value(rows), rows.scales.double().repeat_interleave(128, -1)[:, :y.shape[1]]
    bound = torch.maximum(y.abs() * 2.0 ** -4, scale * 2.0 ** -10) * 1.0001 + y.abs() * slack
    assert bool(((got - y).abs() <= bound).all())
    # and no scale is larger than its block needs
    top = torch.nn.functional.pad(y.abs(), (0, -y.shape[1] % 128)).unflatten(-1, (-1, 128)).amax(-1)
    used = rows.scales.double()[:, :top.shape[1]]
    assert bool((top * (1 + slack) >= 224.0 * used)[used > 2.0 ** -126].all()) and bool((top <= 448.0 * used * (1 + slack)).all())


# ------------------------------------------------------------------------------------------------- rows

@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,K", [(1, 16), (3, 112), (2, 128), (5, 144), (7, 512), (2, 528), (1, 2048), (33, 2064), (4, 14336), (1, 20000), (0, 256)])
def test_rows(ops, dtype, T, K):
    x = uneven(T, K, dtype, seed=T + K)
    same_rows(ops.quantize_fp8(x), x)


@pytest.mark.parametrize("dtype", TYPES)
def test_rows_of_every_size_and_kind(ops, dtype):
    """Every finite magnitude that a block may lead with, zeros, and what is not finite."""
    e = torch.arange(-140, 128, device="cuda", dtype=torch.float64)
    x = rand((e.numel(), 272), seed=3).double() * torch.exp2(e)[:, None]
    x = x.clamp(-3.3e38, 3.3e38).to(dtype)
    x[5] = 0.0
    x[6, :128] = -0.0
    x[7, 3], x[8, 130], x[9, 131], x[10, 270] = math.inf, -math.inf, math.nan, math.inf
    x[11] = math.nan
    x[12, :128] = 448.0
    x[13, :128] = 1.0
    x[13, 0] = 450.0
    same_rows(ops.quantize_fp8(x), x)


def test_ties_and_borders(ops):
    """Numbers halfway between two neighbours go to the even one, whatever the scale."""
    codes = torch.arange(0, 127, device="cuda", dtype=torch.uint8).view(torch.float8_e4m3fn).float()
    half = torch.cat([codes, (codes[1:] + codes[:-1]) / 2])
    half = torch.cat([half, -half, torch.full((-2 * half.numel() % 128,), 3.0, device="cuda")]).reshape(-1, 1)
    rows = torch.cat([half.repeat(1, 127), torch.full_like(half, 448.0)], 1)        # the block's scale is one
    rows = torch.cat([rows, rows * 2.0 ** -60, rows * 2.0 ** 70], 1)
    same_rows(ops.quantize_fp8(rows), rows)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,K,splits", [(1, 16, 1), (2, 2048, 1), (8, 4096, 3), (3, 8208, 1), (2, 16384, 1), (1, 32768, 2), (300, 1040, 1), (0, 64, 1)])
def test_norm(ops, dtype, T, K, splits):
    splits = splits if dtype == torch.float32 else 1         # (partial sums are float32)
    h, w = uneven(T, K, seed=1), 1.0 + 0.3 * rand((K,), seed=2)
    delta = rand((splits, T, K) if splits > 1 else (T, K), dtype, seed=4)
    want_h = h.double() + (delta.double().sum(0) if splits > 1 else delta.double())
    rows = ops.rmsnorm_fp8(h, delta, w, 1e-5)
    # a sum of splits + 1 numbers: an error of half a step each, of at most the sum of magnitudes
    assert bool(((h.double() - want_h).abs() <= (splits + 1) * 2.0 ** -24 * (want_h.abs() + (delta.double().abs().sum(0) if splits > 1 else delta.double().abs()) * splits + 1e-30)).all())
    x = h.double()
    y = x / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-5) * w.double()
    # squares and their sum (32 terms a thread at most, then 10 sums in a tree), a root, a quotient, two products: below 64 half steps
    near_rows(rows, y, 64 * 2.0 ** -24)


@pytest.mark.parametrize("T,K", [(591, 4096), (592, 4096), (592, 16), (700, 2032), (593, 2064), (600, 4112), (595, 8192), (600, 8208)])
def test_norm_of_many_rows(ops, T, K):
    """Both sides of the number of rows and of the widths from which CTAs are smaller; bounds as above (32 terms a thread, 8 sums in a tree)."""
    h, w, delta = uneven(T, K, seed=1), 1.0 + 0.3 * rand((K,), seed=2), rand((T, K), torch.bfloat16, seed=4)
    want_h = h.double() + delta.double()
    rows = ops.rmsnorm_fp8(h, delta, w, 1e-5)
    assert bool(((h.double() - want_h).abs() <= 2.0 ** -24 * (want_h.abs() + 1e-30) * (1 + 2.0 ** -20)).all())
    x = h.double()
    near_rows(rows, x / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-5) * w.double(), 64 * 2.0 ** -24)


def test_norm_without_a_delta_leaves_the_stream(ops):
    h, w = uneven(5, 512, seed=1), 1.0 + 0.3 * rand((512,), seed=2)
    before = h.clone()
    rows = ops.rmsnorm_fp8(h, None, w, 1e-6)
    assert torch.equal(h, before)
    x = h.double()
    near_rows(rows, x / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-6) * w.double(), 64 * 2.0 ** -24)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind,gated", [("silu", True), ("silu", False), ("gelu_tanh", True), ("gelu", False), ("relu2", False), ("relu2", True), ("clamped_swish", True)])
@pytest.mark.parametrize("T,K", [(1, 16), (9, 2048), (70, 4112), (0, 128)])
def test_activation(ops, dtype, kind, gated, T, K):
    params = (3.0, 1.7, 1.0) if kind == "clamped_swish" else None
    u = rand((T, 2 * K if gated else K), dtype, seed=K, scale=2.0)
    rows = ops.activation_fp8(u, kind, gated=gated, act_params=params)
    y = plain.act(u.double(), kind, gated, params)
    # exponentials are off by 2 units and 2^-22 of their argument (at most 17 here), tanh and erf by some 2^-22 of one; where such a
    # sum cancels (gelu far below zero) the error is that much of the argument itself, which the block's scale bounds from above
    got, scale = plain.value(rows), rows.scales.double().repeat_interleave(128, -1)[:, :K]
    slack = 2.0 ** -18
    reach = u.double()[:, :K].abs() * (u.double()[:, K:].abs() + 1.0 if gated else 1.0) * 2.0 ** -21
    bound = torch.maximum(y.abs() * 2.0 ** -4, scale * 2.0 ** -10) * 1.0001 + y.abs() * slack + reach
    assert bool(((got - y).abs() <= bound).all())


def test_activation_keeps_what_is_not_a_number(ops):
    for kind, gated in (("silu", True), ("gelu", False), ("relu2", False), ("clamped_swish", True)):
        u = rand((3, 256), seed=1)
        u[1, 5] = math.nan
        rows = ops.activation_fp8(u, kind, gated=gated, act_params=(2.0, 1.0, 0.0) if gated and kind == "clamped_swish" else None)
        bad = torch.isnan(plain.value(rows))
        assert bad.nonzero().tolist() == [[1, 5]]


# ------------------------------------------------------------------------------------------------- products

def check_product(got, x, w, out_dtype):
    """float32 sums: every product and scaling is exact; the tensor cores' sums are held to 2^-22 of the sum of magnitudes for every
    instruction's sum of 32 (their own rounding, twice a float32's step), then the result's own rounding."""
    a, b = plain.value(x), plain.value(w)
    want, size = a @ b.T, a.abs() @ b.abs().T
    K = a.shape[1]
    bound = size * (K / 32 + 4) * 2.0 ** -24 + want.abs() * (torch.finfo(out_dtype).eps / 2 * 1.001) + 1e-30
    assert got.shape == want.shape and got.dtype == out_dtype
    assert bool(((got.double() - want).abs() <= bound).all()), float(((got.double() - want).abs() / bound).max())


SIZES = [(1, 128, 128), (16, 128, 512), (3, 16, 16), (5, 130, 144), (17, 200, 640), (64, 4096, 4096), (8, 28672, 256), (1, 6144, 2048), (100, 264, 1040),
         (128, 256, 2048), (129, 257, 528), (240, 512, 512), (241, 384, 528), (300, 1000, 4112), (3, 512, 2064), (500, 2048, 8192), (2048, 640, 512), (77, 1, 256), (33, 7, 14336)]


@pytest.mark.parametrize("impl", ["single", "pair", "split", "auto"])
@pytest.mark.parametrize("M,N,K", SIZES)
def test_product(ops, M, N, K, impl):
    x, w = held(uneven(M, K, seed=M)), held(rand((N, K), seed=N + 1, scale=K ** -0.5))
    check_product(ops.linear_fp8(x, w, impl=impl), x, w, torch.bfloat16)
    check_product(ops.linear_fp8(x, w, out_dtype=torch.float32, impl=impl), x, w, torch.float32)
    ops.check_status()


def test_many_units_to_a_cta(ops):
    """More units than CTAs several times over: accumulators, stages and scales go round; calls behind one another without a wait."""
    x, w = held(uneven(1450, 1040, seed=3)), held(rand((9000, 1040), seed=4, scale=1040 ** -0.5))
    runs = {impl: [ops.linear_fp8(x, w, torch.float32, impl=impl) for _ in range(6)] for impl in ("single", "pair")}
    ops.check_status()
    check_product(runs["pair"][0], x, w, torch.float32)
    for impl, outs in runs.items():
        assert all(torch.equal(o, runs["pair"][0]) for o in outs), impl


def test_what_is_not_finite_stays_in_its_row(ops):
    x, w = uneven(40, 640, seed=1), rand((300, 640), seed=2)
    clean = ops.linear_fp8(held(x), held(w))
    x[3, 200], x[17, 0], w[130, 639] = math.nan, math.inf, -math.inf
    got = ops.linear_fp8(x, held(w))
    bad = torch.zeros_like(got, dtype=torch.bool)
    bad[3], bad[17], bad[:, 130] = True, True, True
    assert torch.equal(torch.isnan(got), bad)
    # (the blocks that held them have scales of their other numbers: rows without them keep their bits)
    assert torch.equal(got[~bad], clean[~bad])


@pytest.mark.parametrize("impl", ["single", "pair", "split"])
def test_few_rows_are_the_first_of_more(ops, impl):
    """Products of 1 to 15 rows, behind products of rows that are not numbers (which stay in shared memory): the bits of the first of 16."""
    w, x = held(rand((640, 2064), seed=1, scale=1 / 32)), held(uneven(16, 2064, seed=2))
    poison = held(torch.full((240, 2064), math.nan, device="cuda"))
    want = ops.linear_fp8(x, w, torch.float32, impl=impl)
    acted = None if impl == "split" else ops.linear_activation_fp8(x, w, "silu", gated=impl == "pair", impl=impl)
    for M in range(1, 16):
        ops.linear_fp8(poison, w, impl="pair")
        ops.linear_fp8(poison[:16], w, impl=impl)
        assert torch.equal(ops.linear_fp8(x[:M], w, torch.float32, impl=impl), want[:M])
        if acted is not None:
            ops.linear_fp8(poison, w, impl="pair")
            got = ops.linear_activation_fp8(x[:M], w, "silu", gated=impl == "pair", impl=impl)
            assert torch.equal(got.codes.view(torch.uint8), acted.codes[:M].view(torch.uint8))
            assert torch.equal(got.scales.view(torch.uint8), acted.scales[:M].view(torch.uint8))
    ops.check_status()


@pytest.mark.parametrize("dtype", TYPES)
def test_product_of_rows_that_come_unheld(ops, dtype):
    x, w = uneven(21, 1040, dtype, seed=5), held(rand((512, 1040), seed=6))
    assert torch.equal(ops.linear_fp8(x, w), ops.linear_fp8(held(x), w))


def test_rows_of_all_scales(ops):
    """Scales from 2^-60 to 2^60 on either side, block by block."""
    e = torch.tensor([-60, 0, 30, -30, 60], device="cuda")
    x = rand((9, 640), seed=1) * torch.exp2(e.float()).repeat_interleave(128)
    w = rand((200, 640), seed=2) * torch.exp2(-e.float()).repeat_interleave(128)
    check_product(ops.linear_fp8(held(x), held(w), torch.float32), held(x), held(w), torch.float32)


@pytest.mark.parametrize("impl", ["single", "pair"])
@pytest.mark.parametrize("kind,gated", [("silu", True), ("silu", False), ("gelu_tanh", True), ("gelu_tanh", False), ("gelu", False), ("gelu", True),
                                        ("relu2", False), ("relu2", True), ("clamped_swish", True)])
@pytest.mark.parametrize("M,hidden,K", [(1, 16, 64), (9, 144, 528), (65, 1040, 256), (250, 384, 1040), (500, 4112, 640)])
def test_product_behind_an_activation(ops, M, hidden, K, kind, gated, impl):
    if gated:
        impl = "auto"                   # (128 hidden numbers lie on a pair)
    params = (3.0, 1.7, 1.0) if kind == "clamped_swish" else None
    x, w = held(uneven(M, K, seed=M)), held(rand((hidden * (2 if gated else 1), K), seed=hidden, scale=K ** -0.5))
    rows = ops.linear_activation_fp8(x, w, kind, gated=gated, act_params=params, impl=impl)
    ops.check_status()
    y, dy = plain.activated(plain.value(x), plain.value(w), kind, gated, params)
    assert rows.shape == (M, hidden) and rows.scales.shape == (M, plain.pitch(hidden))
    assert bool(((plain.value(rows) - plain.stands_for(y)).abs() <= plain.moved(y, dy)).all())
    e = plain.hold(y)[1]
    assert bool((rows.scales.view(torch.uint8)[:, e.shape[1]:] == 0).all())
    # a scale is the format's, or its neighbour where the error reaches the border
    off = (rows.scales.view(torch.uint8)[:, :e.shape[1]].double() - (e + 127)).abs()
    assert bool((off <= 1).all()) and float((off > 0).double().mean()) < 0.01 + 2.0 / off.numel()


def test_product_behind_an_activation_keeps_what_is_not_a_number(ops):
    x, w = uneven(40, 640, seed=1), rand((512, 640), seed=2)
    x[3, 200], w[130, 639] = math.nan, math.inf
    for gated in (False, True):
        bad = torch.isnan(plain.value(ops.linear_activation_fp8(held(x), held(w), "silu", gated=gated)))
        want = torch.zeros_like(bad)
        want[3], want[:, 130] = True, True
        assert torch.equal(bad, want)


# ------------------------------------------------------------------------------------------------- experts

def routed(T, E, top, seed, skew=1.0):
    score = rand((T, E), seed=seed) + skew * rand((E,), seed=seed + 1)
    best, chosen = torch.topk(score, top, dim=-1)
    return chosen.int().contiguous(), torch.softmax(best, -1).contiguous()


def check_experts(ops, T, E, top, dim, hidden, kind, gated, dtype, params=None, chosen=None, seed=0, impl="auto"):
    picked, share = routed(T, E, top, seed)
    chosen = picked if chosen is None else chosen
    x = uneven(T, dim, dtype, seed=seed + 2)
    up = held(rand((E, hidden * (2 if gated else 1), dim), seed=seed + 3, scale=dim ** -0.5))
    down = held(rand((E, dim, hidden), seed=seed + 4, scale=hidden ** -0.5))
    got = ops.moe_experts_fp8(x, chosen, share, up, down, activation=kind, gated=gated, act_params=params, impl=impl)
    ops.check_status()
    want = plain.experts(x, chosen, share, plain.value(up), plain.value(down), kind, gated, params)
    assert got.shape == x.shape and got.dtype == dtype
    # a number of every result, by arithmetic (a bound on whole rows that went by how rare borders are did not hold for rows which one
    # hidden number makes up): float32's errors, the borders that they reach, and the result's own roundings
    bound = plain.experts_bound(x, chosen, share, plain.value(up), plain.value(down), kind, gated, params, torch.finfo(dtype).eps / 2 * 1.01)
    assert bool(((got.double() - want).abs() <= bound + 1e-30).all()), float(((got.double() - want).abs() / (bound + 1e-30)).max())
    return got, (x, chosen, share, up, down)


@pytest.mark.parametrize("impl", ["single", "pair"])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,E,top,dim,hidden,kind,gated", [
    (1, 4, 1, 16, 16, "silu", True), (1, 8, 2, 256, 128, "relu2", False), (3, 8, 8, 144, 272, "gelu", False), (8, 32, 4, 512, 896, "relu2", False),
    (8, 32, 4, 512, 896, "silu", True), (65, 16, 4, 1040, 144, "clamped_swish", True), (300, 8, 2, 640, 512, "gelu_tanh", True),
    (700, 4, 2, 256, 1040, "silu", True), (1000, 16, 4, 512, 3584, "silu", True), (40, 64, 1, 528, 400, "relu2", False), (0, 4, 2, 128, 128, "silu", True)])
def test_experts(ops, dtype, T, E, top, dim, hidden, kind, gated, impl):
    check_experts(ops, T, E, top, dim, hidden, kind, gated, dtype, impl=impl, params=(3.0, 1.7, 1.0) if kind == "clamped_swish" else None)


def test_all_tokens_to_one_expert(ops):
    """One expert has every row, many tiles of it, and the others none."""
    chosen = torch.full((600, 1), 5, dtype=torch.int32, device="cuda")
    check_experts(ops, 600, 16, 1, 256, 256, "silu", True, torch.bfloat16, chosen=chosen)


def test_the_same_expert_twice(ops):
    chosen = torch.tensor([[2, 2], [1, 2], [0, 0], [3, 1]], dtype=torch.int32, device="cuda")
    check_experts(ops, 4, 4, 2, 256, 384, "relu2", False, torch.bfloat16, chosen=chosen)


def test_a_token_does_not_depend_on_the_batch(ops):
    got, (x, chosen, share, up, down) = check_experts(ops, 50, 8, 2, 512, 256, "silu", True, torch.bfloat16)
    for t in (0, 17, 49):
        alone = ops.moe_experts_fp8(x[t:t + 1], chosen[t:t + 1], share[t:t + 1], up, down, activation="silu", gated=True)
        assert torch.equal(alone[0], got[t])


@pytest.mark.parametrize("splits", [0, 1, 3])
def test_experts_beside_a_shared_one(ops, splits):
    got, (x, chosen, share, up, down) = check_experts(ops, 20, 8, 2, 512, 256, "relu2", False, torch.bfloat16)
    shared = rand((splits, 20, 512) if splits else (20, 512), torch.float32 if splits else torch.bfloat16, seed=9)
    gate = torch.rand(20, device="cuda")
    both = ops.moe_experts_fp8(x, chosen, share, up, down, activation="relu2", shared=shared, shared_gate=gate)
    extra = (shared.double().sum(0) if splits else shared.double()) * gate.double()[:, None]
    want = plain.experts(x, chosen, share, plain.value(up), plain.value(down), "relu2") + extra
    # the same bounds, of the two terms' sizes
    off = (both.double() - want).norm(dim=-1)
    assert bool((off <= (2.0 ** -10 + 1.5 * 2.0 ** -7) * (got.double().norm(dim=-1) + extra.norm(dim=-1))).all())
