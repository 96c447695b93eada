"""The 8-bit rows' format in PyTorch against its definition in 64 bits, and what the calls refuse (on the host)."""

import math

import pytest
import torch

import fp8_plain as plain
from torchllms_b200.weights.fp8 import CODES, SCALES, Fp8Rows, check_width, decode, encode, scale_pitch


def rows(T, K, seed=0):
    g = torch.Generator().manual_seed(seed)
    return torch.randn((T, K), generator=g) * torch.exp(1.5 * torch.randn((K,), generator=g))


@pytest.mark.parametrize("K", [16, 112, 128, 144, 512, 528, 2064])
def test_encode_holds_what_the_definition_says(K):
    x = rows(20, K, K)
    x[1] = 0.0
    x[2, 0], x[3, 5], x[4, K - 1] = math.inf, math.nan, -math.inf
    x[5] *= 1e-38
    x[6] = (x[6].double() * 1e37).clamp(-3e38, 3e38).float()
    codes, scales = encode(x)
    assert codes.dtype == CODES and scales.dtype == SCALES and codes.shape == x.shape and scales.shape == (20, plain.pitch(K)) == (20, scale_pitch(K))
    held, e = plain.hold(x)
    assert torch.equal(codes.double().nan_to_num(777.0), held.nan_to_num(777.0))
    byte = torch.zeros(scales.shape, dtype=torch.uint8)
    byte[:, :e.shape[1]] = (e + 127).to(torch.uint8)
    assert torch.equal(scales.view(torch.uint8), byte)
    assert torch.equal(decode(codes, scales).double().nan_to_num(7.0), plain.value(Fp8Rows(codes, scales)).float().double().nan_to_num(7.0))


def test_a_second_encoding_changes_nothing():
    x = Fp8Rows(*encode(rows(8, 640, 3))).dequantize()
    codes, scales = encode(x)
    assert torch.equal(decode(codes, scales), x)


def test_error_is_half_a_step():
    x = rows(50, 1024, 4)
    r = Fp8Rows(*encode(x))
    scale = r.scales.float().repeat_interleave(128, -1)
    assert bool(((r.dequantize() - x).abs() <= torch.maximum(x.abs() * 2.0 ** -4, scale * 2.0 ** -10)).all())


def test_experts_and_views():
    x = rows(24, 272, 5).reshape(4, 6, 272)
    r = Fp8Rows(*encode(x))
    assert r.shape == (4, 6, 272) and r.scales.shape == (4, 6, 4) and r.nbytes() == 4 * 6 * 276
    part = r[1:3]
    assert torch.equal(part.dequantize(), r.dequantize()[1:3]) and part.codes.data_ptr() == r.codes[1:].data_ptr()


@pytest.mark.parametrize("K", [0, 8, 100, 130])
def test_widths_that_are_refused(K):
    with pytest.raises(ValueError):
        check_width(K)


def bare_ops():
    """The front end without a GPU behind it: what it refuses, it refuses before anything is launched."""
    from torchllms_b200.kernels.native import NativeOps
    class Nothing:                       # (the C++ front end answers so where something does not fit)
        rows = norm = product = act_product = experts = staticmethod(lambda *args: None)
    ops = object.__new__(NativeOps)
    ops._profile, ops.launches, ops._status_at, ops._fp8 = None, 0, 1, Nothing
    return ops


def test_calls_refuse_the_host():
    from torchllms_b200.kernels.native import KernelError
    ops, x = bare_ops(), rows(4, 256)
    w = Fp8Rows(*encode(rows(32, 256)))
    for call in (lambda: ops.quantize_fp8(x), lambda: ops.activation_fp8(x, "silu"), lambda: ops.rmsnorm_fp8(x, None, x[0], 1e-5),
                 lambda: ops.linear_fp8(x, w), lambda: ops.linear_fp8(w, w), lambda: ops.linear_fp8(w, x), lambda: ops.linear_activation_fp8(w, w, "silu"),
                 lambda: ops.moe_experts_fp8(x, torch.zeros((4, 1), dtype=torch.int32), torch.ones((4, 1)), w, w, activation="silu")):
        with pytest.raises(KernelError):
            call()
    with pytest.raises(KernelError, match="unknown activation"):
        ops.activation_fp8(x, "swish")
    with pytest.raises(KernelError, match="clamped"):
        ops.activation_fp8(x, "clamped_swish")
    assert ops.launches == 0


def test_sizes_at_the_end_of_an_int_are_refused():
    """The products' entries say so before they reckon with them, or ask a device anything."""
    import ctypes
    from torchllms_b200.kernels.build import compile_library
    lib = ctypes.CDLL(str(compile_library("gemm_fp8")))
    some, status = ctypes.c_void_p(1 << 20), (ctypes.c_int * 1)()
    end = 2 ** 31 - 1
    i, f, at = ctypes.c_int, ctypes.c_float, ctypes.byref(status)
    for M, N in ((end, 16), (1, end), (2 ** 31 - 255, 16)):
        for form in range(4):
            assert lib.tl_gemm_fp8(some, some, some, some, some, i(0), i(M), i(N), i(16), i(form), at, None) != 0
    for form in range(3):
        assert lib.tl_gemm_fp8_act(some, some, some, some, some, some, i(end), i(16), i(16), i(0), i(0), f(0), f(0), f(0), i(1), None, i(0), i(form), at,
                                   None) != 0
        assert lib.tl_gemm_fp8_experts(some, some, some, some, some, i(0), i(end), i(16), i(16), i(2), some, i(1), i(form), at, None) != 0
    assert status[0] == 0
