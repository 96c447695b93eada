// Keys and values held in 4 bits: the numbers, their scales, and where they lie.
//
// Sixteen neighbouring coordinates of a token's key (or value) of one head are a group: 4-bit numbers, a sign and one of
// 0, 0.5, 1, 1.5, 2, 3, 4, 6 (E2M1), and one byte of scale, 5 bits of exponent and 3 of mantissa, no sign:
//     scale(E, M) = M 2^-17 for E = 0, else (8 + M) 2^(E - 18).
// With a = max |x| of the group, scale = a / 6 rounded to nearest (ties to even) and at most 10240, a number is x / scale
// rounded to nearest (ties to the even code), at most 6.  A group that holds a number which is not finite has the scale
// byte 255 and reads as NaN throughout, so that such a number does not vanish; attention gives it to the rows that see its token, and to
// no others.  A group below 6 * 2^-18 reads as zeros.
//
// What that choice buys the readers: the scale's byte shifted left by 7 is the float16 with its value, and a number times
// its scale has 2 + 4 significant bits and lies between 2^-18 and 61440, so it IS a float16.  Attention over the cache
// multiplies exactly the cached numbers on the float16 tensor cores; nothing is rounded on the way out of the cache.
//
// Sixteen tokens of a head are a record of 9 * head_dim bytes (144 a token at head_dim 128, k and v; bfloat16 takes 512): 16
// rows of head_dim / 2 bytes, coordinate 2 i in the low half of byte i, then 16 rows of head_dim / 16 scales.  A head's part
// of a page is page_size / 16 records, one behind the other, so a reader fetches whole records whatever the page size.
#pragma once

#include "common.cuh"
#include <cuda_fp16.h>

constexpr int FP4_GROUP = 16;          // numbers that share a scale
constexpr int FP4_RECORD = 16;         // tokens of a record
constexpr int FP4_TOP_SCALE = 226;     // the scale byte of 10240
constexpr int FP4_NAN_SCALE = 255;

__host__ __device__ constexpr int fp4_record_bytes(int head_dim) { return 9 * head_dim; }

// Eight numbers (a 32-bit word) as float16 pairs, unscaled.
__device__ __forceinline__ void fp4_unpack(unsigned w, __half2 (&r)[4]) {
    unsigned u[4];
    asm("{.reg .b8 a, b, c, d;\n\tmov.b32 {a, b, c, d}, %4;\n\tcvt.rn.f16x2.e2m1x2 %0, a;\n\tcvt.rn.f16x2.e2m1x2 %1, b;\n\t"
        "cvt.rn.f16x2.e2m1x2 %2, c;\n\tcvt.rn.f16x2.e2m1x2 %3, d;\n\t}"
        : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]) : "r"(w));
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = *reinterpret_cast<__half2*>(&u[i]);
}
// Two numbers (a byte).  (Through a word of four such bytes: for a byte that was widened with zeros, nvcc 12.9 gave zeros.)
__device__ __forceinline__ __half2 fp4_unpack2(unsigned byte) {
    __half2 r[4];
    fp4_unpack(byte * 0x01010101u, r);
    return r[0];
}
// A scale's byte as a pair of float16.
__device__ __forceinline__ __half2 fp4_scale2(unsigned byte) {
    const unsigned u = byte * 0x00800080u;
    return *reinterpret_cast<const __half2*>(&u);
}
__device__ __forceinline__ float fp4_scale(unsigned byte) { return __half2float(__ushort_as_half((unsigned short)(byte << 7))); }

// The scale's byte for a group whose largest magnitude has these bits (of a float32 without its sign).
__device__ __forceinline__ unsigned fp4_scale_byte(unsigned top_bits) {
    if (top_bits >= 0x7f800000u) return FP4_NAN_SCALE;
    const float want = __fdiv_rn(__uint_as_float(top_bits), 6.f);
    if (want < 6.103515625e-05f) return (unsigned)__float2int_rn(want * 131072.f);      // below 2^-14: multiples of 2^-17
    const unsigned bits = __float_as_uint(want);
    const int byte = (int)((bits + 0x7ffffu + ((bits >> 20) & 1u)) >> 20) - (112 << 3);
    return (unsigned)min(byte, FP4_TOP_SCALE);
}
// Two numbers, already divided by their scale, as a byte (`lo` in its low half).
__device__ __forceinline__ unsigned fp4_pack2(float lo, float hi) {
    unsigned short v;
    asm("{.reg .b8 a;\n\tcvt.rn.satfinite.e2m1x2.f32 a, %1, %2;\n\tmov.b16 %0, {a, 0};\n\t}" : "=h"(v) : "f"(hi), "f"(lo));
    return v;
}
// Eight numbers of a group under the scale with this byte.  The quotients are those of IEEE division (one that lies exactly between
// two codes, and bfloat16 inputs have many, must not be pushed off it): with the reciprocal rounded to nearest, a quotient that
// is off by an ulp at most is put right by its remainder (Markstein, 1990), three multiply-adds instead of a division.
__device__ __forceinline__ unsigned fp4_pack8(const float (&x)[8], unsigned byte) {
    if (byte == 0u || byte == (unsigned)FP4_NAN_SCALE) return 0u;
    const float scale = fp4_scale(byte), inverse = __frcp_rn(scale);
    unsigned w = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        float q[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const float y = x[2 * i + e] * inverse;
            // (far above the largest number the remainder may overflow: saturated either way)
            q[e] = fabsf(y) < 64.f ? fmaf(fmaf(-y, scale, x[2 * i + e]), inverse, y) : y;
        }
        w |= fp4_pack2(q[0], q[1]) << (8 * i);
    }
    return w;
}

// Attention: whether all places of a step stay within 32 bits, also with a tile added or a window taken off.  (A row's place is below zero, down to
// minus max_q_len, where a request is shorter than its new tokens.)
static inline bool fp4_places_fit(int table_cols, int page_size, int max_q_len) {
    return (double)table_cols * page_size + (double)max_q_len + 4096.0 < 2147483648.0;
}
// The window as the kernels take it, 0 for none: one that holds every key that a table can name is none.
static inline int fp4_window(int window, int table_cols, int page_size) {
    return window > 0 && (long long)window < (long long)table_cols * page_size ? window : 0;
}

// Where a token of a head lies: its row of numbers and its row of scales.
struct Fp4Place {
    long long codes, scales;
};
__device__ __forceinline__ Fp4Place fp4_place(long long page, int slot, int head, int n_heads, int page_size, int head_dim) {
    const long long record = (page * n_heads + head) * (page_size / FP4_RECORD) + slot / FP4_RECORD;
    const long long at = record * fp4_record_bytes(head_dim);
    const int row = slot % FP4_RECORD;
    return {at + row * (head_dim / 2), at + FP4_RECORD * (head_dim / 2) + row * (head_dim / FP4_GROUP)};
}
