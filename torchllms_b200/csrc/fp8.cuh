// Rows of numbers in 8 bits, the kernels' side (the format in PyTorch: weights/fp8.py).
//
// 128 neighbouring numbers of a row share a scale 2^e, e the least integer with a <= 448 * 2^e where a is their largest finite
// magnitude, at least -126 and at most 120; a number is held as E4M3 of x * 2^-e, rounded to nearest (ties to even).  The scale is
// a power of two, so the division is exact and the only rounding is that to E4M3's four significant bits; and it is the
// E8M0 byte e + 127 that the block-scaled tensor-core instructions multiply by.  What is not finite is held as NaN.
#pragma once
#include "common.cuh"
#include <math.h>

constexpr int FP8_BLOCK = 128;       // numbers that share a scale

// bytes of scales a row of K numbers has: one for every 128, in whole words (the places behind the last are 0)
__host__ __device__ __forceinline__ int fp8_scale_pitch(int K) { return 4 * ((K + 511) / 512); }

// the exponent for a largest magnitude given by its bits (finite, sign cleared): 448 = 1.75 * 2^8
__device__ __forceinline__ int fp8_exponent(unsigned top_bits) {
    const int e = (int)(top_bits >> 23) - 135 + ((top_bits & 0x7fffffu) > 0x600000u ? 1 : 0);
    return e < -126 ? -126 : e;
}
__device__ __forceinline__ float fp8_inverse(int e) { return __int_as_float((127 - e) << 23); }

// two numbers, already divided by their scale, as two bytes (the first one low); infinities must not get here
__device__ __forceinline__ unsigned fp8_pack2(float lo, float hi) {
    unsigned short r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
    return r;
}

// Eight numbers of a 128-number block that lies on 16 lanes (the other half warp has a block of its own): the scale's exponent
// (the same on all 16 lanes) and the eight bytes.  Lanes behind the end of the row bring zeros.  Whole warps call it.
__device__ __forceinline__ int fp8_encode8(const float (&v)[8], uint2& bytes) {
    unsigned top = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(v[i]) & 0x7fffffffu);
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
    const bool odd = top >= 0x7f800000u;                  // (16 lanes alike) something is not finite
    if (__any_sync(0xffffffffu, odd)) {
        unsigned fine = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const unsigned b = __float_as_uint(v[i]) & 0x7fffffffu;
            if (b < 0x7f800000u) fine = max(fine, b);
        }
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) fine = max(fine, __shfl_xor_sync(0xffffffffu, fine, o));
        top = fine;
    }
    const int e = fp8_exponent(top);
    const float inv = fp8_inverse(e);
    float t[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) t[i] = v[i] * inv;
    if (odd) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if ((__float_as_uint(v[i]) & 0x7f800000u) == 0x7f800000u) t[i] = __int_as_float(0x7fffffff);
    }
    bytes.x = fp8_pack2(t[0], t[1]) | (fp8_pack2(t[2], t[3]) << 16);
    bytes.y = fp8_pack2(t[4], t[5]) | (fp8_pack2(t[6], t[7]) << 16);
    return e;
}

// ---- activations of feed-forwards: the codes and the functions of csrc/moe.cu, in forms that keep their relative error where they vanish
// (a block may hold nothing else, and its scale follows its numbers)
enum : int { FP8_SILU = 0, FP8_GELU_TANH = 1, FP8_RELU2 = 2, FP8_CLAMPED_SWISH = 3, FP8_GELU = 4 };
struct Fp8Gate { float limit, alpha, up_offset; };

// x / (1 + e^-y) by e^-|y|, which is at most 1, so the divisor lies between 1 and 2, where its approximate reciprocal is off by one unit; __expf is
// off by 2 + 1.17 |y| of them (2^-16 at 95): far below the step of E4M3 that follows.
__device__ __forceinline__ float fp8_times_sigmoid(float x, float y) {
    const float e = __expf(-fabsf(y));
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.f + e));
    return (y < 0.f ? x * e : x) * r;
}
// The normal distribution below -t, for t >= 0: e^(-t^2 / 2) q P(q), q = 1 / (1 + 0.345 t).  P was fitted to Mills' ratio over sqrt(2 pi)
// from 0 to 15 by least squares of the relative error, weighted until its largest was least (2.6e-8; 3e-7 with float32's roundings).  (CUDA's
// normcdff, which does not cancel either: 1,531 rows of gates and ups of 14,336 by gelu 56 us; erff, which does, 34; this 30.)
__device__ __forceinline__ float fp8_normal_tail(float t) {
    float q, p = -0.0279335193f;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(q) : "f"(fmaf(0.345f, t, 1.f)));
    const float c[8] = {0.137620866f, 0.137990683f, 0.117477998f, 0.110766202f, -0.0349472314f, 0.183022812f, -0.267236143f, 0.143238321f};
#pragma unroll
    for (int i = 7; i >= 0; --i) p = fmaf(p, q, c[i]);
    return __expf(-0.5f * t * t) * (p * q);
}
__device__ __forceinline__ float fp8_act(float x, int act) {
    if (act == FP8_SILU) return fp8_times_sigmoid(x, x);
    if (act == FP8_GELU_TANH) return fp8_times_sigmoid(x, 1.5957691216057308f * (x + 0.044715f * x * x * x));      // (1 + tanh y) / 2 = sigmoid(2 y)
    if (act == FP8_GELU) {                       // (1 + erf(x / sqrt 2)) / 2, without the difference that cancels below 0
        const float p = fp8_normal_tail(fabsf(x));
        return x < 0.f ? x * p : fmaf(-x, p, x);
    }
    const float r = x < 0.f ? 0.f : x;           // (comparisons, not fmaxf: what is not a number stays so)
    return r * r;
}
__device__ __forceinline__ float fp8_gated(float gate, float up, int act, const Fp8Gate& p) {
    if (act == FP8_CLAMPED_SWISH) {
        const float g = gate > p.limit ? p.limit : gate, u = up > p.limit ? p.limit : (up < -p.limit ? -p.limit : up);
        return fp8_times_sigmoid(g, p.alpha * g) * (u + p.up_offset);
    }
    return fp8_act(gate, act) * up;
}
