"""The 8-bit rows' operators where a rounding too many, a value far out or the order of launches would show: each case by itself."""

import pytest
import torch

import fp8_plain as plain
from torchllms_b200.weights.fp8 import Fp8Rows, encode

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from torchllms_b200.kernels import get_ops
    return get_ops()


def rand(shape, dtype=torch.float32, seed=0, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)


def whole(lo, hi, shape, seed):
    return torch.randint(lo, hi + 1, shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda").float()


def held(x):
    return Fp8Rows(*encode(x))


# ------------------------------------------------------------------------------------------------- one rounding

def check_one_rounding(got, x, chosen, share, up, down, extra=None):
    """Small whole numbers, which 8 bits hold as they are, all the way to the experts' results: those are exact in float32, and what is left
    are the weighted sum's errors in float32 (an error of half a step for each of its terms) and one rounding to the result's type."""
    terms = torch.zeros(x.shape, dtype=torch.float64, device="cuda")
    want = torch.zeros_like(terms)
    for k in range(chosen.shape[1]):
        u = torch.einsum("td,thd->th", x.double(), up[chosen[:, k].long()].double())
        z = torch.einsum("th,tdh->td", u.clamp(min=0) ** 2, down[chosen[:, k].long()].double()) * share[:, k, None].double()
        want, terms = want + z, terms + z.abs()
    if extra is not None:
        want, terms = want + extra, terms + extra.abs()
    slack = terms * (chosen.shape[1] + 2) * 2.0 ** -24
    bound = slack + (want.abs() + slack) * (torch.finfo(got.dtype).eps / 2)
    assert bool(((got.double() - want).abs() <= bound).all()), float(((got.double() - want).abs() / (bound + 1e-30)).max())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T,E,top,dim,hidden", [(1, 4, 3, 16, 64), (40, 8, 4, 144, 128), (300, 4, 4, 512, 256), (33, 16, 7, 272, 144)])
def test_experts_results_are_rounded_once(ops, dtype, T, E, top, dim, hidden):
    # (a token's row has one number, and the hidden ones are squares of 0 to 3: all of them numbers of E4M3 under one scale)
    x = torch.zeros((T, dim), device="cuda")
    x[torch.arange(T), whole(0, dim - 1, (T,), 1).long()] = 1.0
    up, down = whole(-1, 3, (E, hidden, dim), 2), whole(-15, 15, (E, dim, hidden), 3)
    chosen = whole(0, E - 1, (T, top), 4).int()
    share = rand((T, top), seed=5)                    # (of either sign: results that cancel keep their experts' errors)
    out = ops.moe_experts_fp8(x.to(dtype), chosen, share, held(up), held(down), activation="relu2")
    check_one_rounding(out, x, chosen, share, up, down)
    gate = torch.rand(T, generator=torch.Generator(device="cuda").manual_seed(7), device="cuda")
    for shared in (rand((T, dim), dtype, seed=6, scale=100.0), rand((2, T, dim), seed=6, scale=100.0)):
        out = ops.moe_experts_fp8(x.to(dtype), chosen, share, held(up), held(down), activation="relu2", shared=shared, shared_gate=gate)
        extra = (shared.double().sum(0) if shared.dim() == 3 else shared.double()) * gate.double()[:, None]
        check_one_rounding(out, x, chosen, share, up, down, extra)
    ops.check_status()


# ------------------------------------------------------------------------------------------------- weights that were made just before

MADE = [("linear", "single"), ("linear", "pair"), ("linear", "split"), ("linear", "auto"), ("act", "single"), ("act", "pair"), ("gated", "auto")]


def made_and_used(ops, kind, impl, weight, x):
    """A weight brought to 8 bits by the kernel in front of the product (held rows), or in front of the rows' kernel (others)."""
    w = ops.quantize_fp8(weight)
    if kind == "linear":
        return ops.linear_fp8(x, w, torch.float32, impl=impl)
    rows = ops.linear_activation_fp8(x, w, "silu", gated=kind == "gated", impl=impl)
    return torch.cat([rows.codes.view(torch.uint8), rows.scales.view(torch.uint8)], 1)


def used_alone(ops, kind, impl, weight, x):
    w = held(weight)
    torch.cuda.synchronize()
    if kind == "linear":
        return ops.linear_fp8(x, w, torch.float32, impl=impl)
    rows = ops.linear_activation_fp8(x, w, "silu", gated=kind == "gated", impl=impl)
    return torch.cat([rows.codes.view(torch.uint8), rows.scales.view(torch.uint8)], 1)


@pytest.mark.parametrize("unheld", [False, True])
@pytest.mark.parametrize("kind,impl", MADE)
@pytest.mark.parametrize("N,K", [(512, 640), (8192, 2048)])
def test_a_weight_made_by_the_kernel_before(ops, N, K, kind, impl, unheld):
    """Other weights from run to run, in the same place of a recorded graph, where nothing stands between the two launches."""
    x = rand((24, K), torch.bfloat16, seed=1)
    x = x if unheld else held(x)
    weights = [rand((N, K), seed=10 + i, scale=K ** -0.5 * 4.0 ** i) for i in range(3)]
    want = [used_alone(ops, kind, impl, w, x) for w in weights]
    place = weights[0].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        made_and_used(ops, kind, impl, place, x)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = [made_and_used(ops, kind, impl, place, x) for _ in range(8)]
    for i in (0, 1, 2, 0, 2, 1):
        place.copy_(weights[i])
        graph.replay()
        assert all(torch.equal(o, want[i]) for o in out)
    for i in range(3):                                   # (the same without a graph, launches queued one behind the other)
        assert all(torch.equal(o, want[i]) for o in [made_and_used(ops, kind, impl, weights[i], x) for _ in range(8)])
    ops.check_status()


def test_rows_times_themselves(ops):
    """The same rows on both sides, straight from the norm that made them."""
    h, w = rand((300, 1040), seed=1), torch.ones(1040, device="cuda")
    rows = ops.rmsnorm_fp8(h, None, w, 1e-5)
    torch.cuda.synchronize()
    want = ops.linear_fp8(rows, rows, torch.float32)
    for _ in range(20):
        rows = ops.rmsnorm_fp8(h, None, w, 1e-5)
        assert torch.equal(ops.linear_fp8(rows, rows, torch.float32), want)
    ops.check_status()


# ------------------------------------------------------------------------------------------------- what CTAs of a cluster send each other

@pytest.mark.parametrize("M", [1, 7, 32])
def test_sums_sent_between_ctas(ops, M):
    """K cut among the CTAs of a cluster, whole numbers: every sum is exact, in every one of many launches one behind the other."""
    x, w = whole(-3, 3, (M, 8192), 1), whole(-3, 3, (640, 8192), 2)
    want = (x.double() @ w.double().T).float()
    xs, ws = held(x), held(w)
    assert all(torch.equal(ops.linear_fp8(xs, ws, torch.float32, impl="split"), want) for _ in range(100))
    ops.check_status()


@pytest.mark.parametrize("M", [3, 200, 481])
def test_magnitudes_sent_between_ctas(ops, M):
    """The largest of 128 gated numbers is now one CTA's, now the other's: scales by the definition, in every launch."""
    hidden, K = 1024, 128
    x = torch.zeros((M, K), device="cuda")
    x[torch.arange(M), torch.arange(M) % K] = 1.0
    # u of column d is 2^(-20 .. 20) in one place of the 128, one beside it: squares of them leave
    up = torch.full((hidden, K), 2.0 ** -24, device="cuda")
    place = whole(0, 127, (hidden // 128, K), 3).long()
    power = torch.exp2(whole(-20, 20, (hidden // 128, K), 4))
    up.view(hidden // 128, 128, K).scatter_(1, place[:, None], power[:, None])
    ws = held(torch.cat([up, up]))
    value = plain.value(ws)[:hidden]
    want = value[:, torch.arange(M, device="cuda") % K].T.clamp(min=0) ** 3            # relu2(g) * u, exact
    codes, e = plain.hold(want)
    for _ in range(50):
        rows = ops.linear_activation_fp8(held(x), ws, "relu2", gated=True)
        assert torch.equal(rows.scales.view(torch.uint8)[:, :e.shape[1]].double(), e + 127)
        assert torch.equal(rows.codes.double(), codes)
    ops.check_status()


# ------------------------------------------------------------------------------------------------- choices that are no experts

def padded(T, E, top, seed):
    """Choices of which some are no experts, with weights that would spoil a sum; one token has no expert at all."""
    chosen, share = whole(0, E - 1, (T, top), seed).int(), rand((T, top), seed=seed + 1).abs()
    real = torch.rand((T, top), generator=torch.Generator(device="cuda").manual_seed(seed + 2), device="cuda") < 0.7
    real[T // 2] = False
    odd = torch.tensor([-1, E, -2 ** 31, 2 ** 31 - 1], dtype=torch.int32, device="cuda")[whole(0, 3, (T, top), seed + 3).long()]
    spoilt = torch.where(whole(0, 1, (T, top), seed + 4) == 1, torch.full_like(share, float("nan")), torch.full_like(share, float("inf")))
    zero = torch.zeros_like(share)
    return torch.where(real, chosen, odd), torch.where(real, share, spoilt), torch.where(real, chosen, torch.zeros_like(chosen)), torch.where(real, share, zero)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T,E,top", [(1, 4, 2), (20, 8, 2), (300, 8, 4), (33, 16, 7)])
def test_choices_that_are_no_experts_add_nothing(ops, dtype, T, E, top):
    chosen, share, instead, nothing = padded(T, E, top, 11)
    x = rand((T, 128), dtype, seed=1)
    up, down = rand((E, 96, 128), dtype, seed=2, scale=0.1), rand((E, 128, 96), dtype, seed=3, scale=0.1)
    shared = rand((T, 128), dtype, seed=4)
    for extra in (None, shared):
        got = ops.moe_experts_fp8(x, chosen, share, held(up), held(down), activation="silu", shared=extra)
        assert torch.equal(got, ops.moe_experts_fp8(x, instead, nothing, held(up), held(down), activation="silu", shared=extra))
        assert torch.equal(got[T // 2], torch.zeros_like(got[0]) if extra is None else shared[T // 2])
        side = down.permute(1, 0, 2).reshape(128, E * 96).contiguous()
        got = ops.moe_experts(x, chosen, share, up, side, activation="silu", shared=extra)
        assert bool(torch.isfinite(got).all())
        assert torch.equal(got[T // 2], torch.zeros_like(got[0]) if extra is None else shared[T // 2])
        if T * top < ops.GROUPED_MIN_PAIRS or dtype == torch.float32:
            assert torch.equal(got, ops.moe_experts(x, instead, nothing, up, side, activation="silu", shared=extra))
    ops.check_status()


def test_no_choice_is_an_expert(ops):
    chosen = torch.full((5, 3), -1, dtype=torch.int32, device="cuda")
    share = torch.full((5, 3), float("nan"), device="cuda")
    up, down = held(rand((4, 32, 128), seed=1)), held(rand((4, 128, 32), seed=2))
    for _ in range(3):
        assert bool((ops.moe_experts_fp8(rand((5, 128), seed=3), chosen, share, up, down, activation="gelu") == 0).all())
    ops.check_status()


def test_layers_of_experts_as_one_matrix_take_padding(ops):
    """The form for few tokens: all experts' hidden rows, a column times its expert's weight."""
    chosen, share, instead, nothing = padded(6, 4, 2, 21)
    keep = nothing != 0
    x, up = rand((6, 128), torch.bfloat16, seed=1), rand((4 * 96, 128), torch.bfloat16, seed=2, scale=0.1)
    got = ops.moe_dense_hidden(x, chosen, share, None, up, n_experts=4, hidden=96, activation="silu")
    weight = torch.zeros((6, 4), device="cuda")
    for t in range(6):
        for k in range(2):
            if keep[t, k]:
                weight[t, int(chosen[t, k])] = share[t, k]
    assert bool(torch.isfinite(got).all()) and bool(((got.view(6, 4, 96) != 0).any(-1) == (weight != 0)).all())


# ------------------------------------------------------------------------------------------------- activations that vanish

def check_far_rows(rows, y, slack):
    """Half a step of E4M3 (2^-4 of the number, 2^-10 of the scale), ``slack`` and a relative 2^-14: exponentials are off by 2 + 1.173 times their
    argument units of 2^-23 (2^-16 at 100), a quotient by two, an argument of 2^-24 of itself three times over shifts them by as much again."""
    got, scale = plain.value(rows), rows.scales.double().repeat_interleave(128, -1)[:, :y.shape[1]]
    bound = torch.maximum(y.abs() * 2.0 ** -4, scale * 2.0 ** -10) * 1.0001 + y.abs() * 2.0 ** -14 + slack
    assert bool(((got - y).abs() <= bound).all()), float(((got - y).abs() / bound).max())
    # scales follow the numbers of their block
    top = torch.nn.functional.pad(y.abs() + 0 * scale, (0, -y.shape[1] % 128)).unflatten(-1, (-1, 128)).amax(-1)
    used = rows.scales.double()[:, :top.shape[1]]
    far = torch.nn.functional.pad(slack, (0, -y.shape[1] % 128)).unflatten(-1, (-1, 128)).amax(-1)
    assert bool((top * (1 + 2.0 ** -14) + far >= 224.0 * used)[used > 2.0 ** -126].all()) and bool((top * (1 - 2.0 ** -14) - far <= 448.0 * used).all())


@pytest.mark.parametrize("kind,lo,hi", [("silu", -100.0, -20.0), ("gelu", -5.5, -3.0), ("gelu_tanh", -5.5, -3.0), ("clamped_swish", -55.0, -10.0)])
def test_activations_of_gates_far_below_zero(ops, kind, lo, hi):
    """Blocks of 128 whose numbers are all of one small size: from gates of nearly the same value, steps apart from row to row."""
    T, K = 400, 256
    params = (1e32, 1.7, 0.0) if kind == "clamped_swish" else None
    gate = torch.linspace(lo, hi, T, device="cuda")[:, None] * (1.0 + 0.001 * torch.rand((T, K), generator=torch.Generator(device="cuda").manual_seed(1), device="cuda"))
    up = rand((T, K), seed=2) * 1e30
    y = plain.act(torch.cat([gate, up], 1).double(), kind, True, params)
    # (an exponential, and its product with the gate, may be below float32's smallest normal number: steps of 2^-149, before the large factor)
    tiny = (gate.double().abs() + 1.0) * up.double().abs() * 2.0 ** -148
    check_far_rows(ops.activation_fp8(torch.cat([gate, up], 1), kind, gated=True, act_params=params), y, tiny)
    if kind != "clamped_swish":
        y = plain.act(gate.double(), kind)
        check_far_rows(ops.activation_fp8(gate, kind), y, (gate.double().abs() + 1.0) * 2.0 ** -148)


@pytest.mark.parametrize("kind,values", [("silu", (-104.0, -96.0, -88.0, -80.0, -36.0, -20.0)), ("gelu", (-5.5, -5.0, -4.5, -4.0, -3.5)),
                                         ("gelu_tanh", (-5.5, -5.0, -4.5, -4.0, -3.5)), ("clamped_swish", (-60.0, -48.0, -22.0, -9.0))])
def test_products_behind_activations_of_gates_far_below_zero(ops, kind, values):
    """The same behind a product: a row of x picks a column of W, whose rows all hold one gate and numbers of E4M3 beside it."""
    params = (2.0 ** 100, 1.75, 0.0) if kind == "clamped_swish" else None
    hidden, K, M = 256, 128, len(values)
    x = torch.zeros((M, K), device="cuda")
    x[torch.arange(M), torch.arange(M)] = 1.0
    up = torch.zeros((hidden, K), device="cuda")
    up[:, :M] = whole(8, 15, (hidden, M), 3) * 2.0 ** 96                 # (four significant bits)
    for m, v in enumerate(values):
        gate = torch.zeros((hidden, K), device="cuda")
        gate[:, m] = v
        w = torch.cat([gate, up])
        u = torch.zeros((M, 2 * hidden), device="cuda", dtype=torch.float64)
        u[m, :hidden] = v
        u[:, hidden:] = plain.value(held(up))[:, :M].T
        y = plain.act(u, kind, True, params)
        slack = (u[:, :hidden].abs() + 1.0) * u[:, hidden:].abs() * 2.0 ** -148
        check_far_rows(ops.linear_activation_fp8(held(x), held(w), kind, gated=True, act_params=params), y, slack)
        if params is None:
            check_far_rows(ops.linear_activation_fp8(held(x), held(gate), kind), plain.act(u[:, :hidden], kind), (u[:, :hidden].abs() + 1.0) * 2.0 ** -148)
    ops.check_status()


# ------------------------------------------------------------------------------------------------- a run of them, recorded

@pytest.mark.parametrize("T", [1, 9, 200])
def test_every_output_of_a_recorded_run(ops, T):
    """Codes, scales, sums and the stream of a replayed run against an eager one's, byte by byte, with other inputs from replay to replay."""
    dim, hidden, E = 512, 640, 8
    w13, w2 = held(rand((2 * hidden, dim), seed=4, scale=dim ** -0.5)), held(rand((dim, hidden), seed=5, scale=hidden ** -0.5))
    up, down = held(rand((E, hidden, dim), seed=6, scale=dim ** -0.5)), held(rand((E, dim, hidden), seed=7, scale=hidden ** -0.5))
    norm = 1.0 + 0.1 * rand((dim,), seed=3)

    def inputs(seed):
        best, chosen = torch.topk(rand((T, E), seed=seed), 2, dim=-1)
        chosen = chosen.int().contiguous()
        chosen[T // 2, 1] = -1                          # (padding)
        return [rand((T, dim), seed=seed + 1), rand((T, dim), torch.bfloat16, seed=seed + 2), chosen, torch.softmax(best, -1).contiguous()]

    def chain(h, delta, chosen, share):
        rows = ops.rmsnorm_fp8(h, delta, norm, 1e-5)
        act = ops.linear_activation_fp8(rows, w13, "silu", gated=True)
        y = ops.linear_fp8(act, w2)
        z = ops.moe_experts_fp8(y, chosen, share, up, down, activation="gelu")
        again = ops.quantize_fp8(z)
        last = ops.activation_fp8(z, "relu2")
        return [t.view(torch.uint8) for r in (rows, act, again, last) for t in (r.codes, r.scales)] + [y, z, h]

    place = [t.clone() for t in inputs(0)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        chain(*[t.clone() for t in place])
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = chain(*place)
    for seed in (0, 30, 60, 30):
        for t, v in zip(place, inputs(seed)):
            t.copy_(v)
        graph.replay()
        want = chain(*inputs(seed))
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    ops.check_status()


@pytest.mark.parametrize("T,E,top", [(700, 4096, 64), (1, 4096, 64), (2000, 3, 64)])
def test_the_most_experts_and_choices(ops, T, E, top):
    """As many experts and choices of a token as there may be: exact results, so that every pair is seen to be placed once."""
    x = torch.zeros((T, 16), device="cuda")
    x[torch.arange(T), whole(0, 15, (T,), 1).long()] = 1.0
    up, down = whole(-1, 3, (E, 16, 16), 2), whole(-15, 15, (E, 16, 16), 3)
    chosen, share = whole(0, E - 1, (T, top), 4).int(), rand((T, top), seed=5)
    check_one_rounding(ops.moe_experts_fp8(x, chosen, share, held(up), held(down), activation="relu2"), x, chosen, share, up, down)
    ops.check_status()


# ------------------------------------------------------------------------------------------------- norms, next to borders

@pytest.mark.parametrize("T,K", [(2048, 4096), (500, 4096), (60, 16384), (40000, 16), (900, 1040)])
def test_norms_are_rounded_once(ops, T, K):
    """Every code and scale is that of the 64-bit row of the stream as it was left: what lies ahead of E4M3's rounding is off by some 2^-42 (eps
    as a float32; all else 2^-47), so one number in 2^37 may stand that close to a border."""
    h, w = rand((T, K), seed=1) * torch.exp(rand((K,), seed=2)), 1.0 + 0.2 * rand((K,), seed=3)
    rows = ops.rmsnorm_fp8(h, rand((T, K), torch.bfloat16, seed=4), w, 1e-5)
    x = h.double()
    codes, e = plain.hold(x / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-5) * w.double())
    assert torch.equal(rows.scales.view(torch.uint8)[:, :e.shape[1]].double(), e + 127)
    assert torch.equal(rows.codes.double(), codes)


def test_norms_of_rows_far_out(ops):
    """Rows whose squares leave float32's range, weights of any size, rows that end a block's scale exactly, rows of one number."""
    T, K = 64, 256
    h = rand((T, K), seed=1) * torch.exp2(torch.linspace(-100, 100, T, device="cuda").round())[:, None]
    w = torch.exp2(whole(-60, 20, (K,), 2)) * (1.0 + whole(0, 7, (K,), 3) / 8)
    h[5], h[6] = 0.0, torch.where(torch.arange(K, device="cuda") == 9, 3.0, 0.0)
    rows = ops.rmsnorm_fp8(h, None, w, 1e-30)
    x = h.double()
    codes, e = plain.hold(x / torch.sqrt((x * x).mean(-1, keepdim=True) + torch.tensor(1e-30, dtype=torch.float32).double()) * w.double())
    assert torch.equal(rows.scales.view(torch.uint8)[:, :e.shape[1]].double(), e + 127)
    assert torch.equal(rows.codes.double(), codes)


def test_norms_keep_what_is_not_finite(ops):
    h, w = rand((6, 256), seed=1), torch.ones(256, device="cuda")
    h[1, 3], h[2, 200], w[7] = float("nan"), float("inf"), float("inf")
    bad = torch.isnan(plain.value(ops.rmsnorm_fp8(h, None, w, 1e-5)))
    want = torch.zeros_like(bad)
    want[1], want[:, 7] = True, True
    want[2, 200] = True                       # (an infinite row: the others are divided by infinity)
    assert torch.equal(bad, want)
