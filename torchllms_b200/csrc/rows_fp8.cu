// Rows into 8 bits (format: fp8.cuh): as they are, behind a residual sum and an RMS norm, behind an activation.
//
// rows:  codes, scales of x.
// norm:  x = h + delta, h <- x, in float32;  y = x * rsqrt(mean(x^2) + eps) * w;  codes, scales of y.
//        (RMSNorm, torchllms/models/networks.py:195-200: the rows go straight to 8 bits, rounded once.)
// act:   y = act(u), or act(g) * u of the halves of a row, in float32;  codes, scales of y.
//
// All three read every number once and write a byte for it: bandwidth is what bounds them, or the launch where rows are few.
// A block of 128 numbers lies on 16 lanes, eight numbers each: 16 bytes a load in bfloat16, 128 contiguous bytes of codes
// a half warp, its largest magnitude in four exchanges.
#include "fp8.cuh"

namespace {

constexpr int ROWS_THREADS = 256;

__device__ __forceinline__ void load8(const float* p, float (&v)[8]) {
    const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}
__device__ __forceinline__ void load8(const __nv_bfloat16* p, float (&v)[8]) {
    const uint4 r = *reinterpret_cast<const uint4*>(p);
    const unsigned w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        v[2 * i] = __uint_as_float(w[i] << 16);
        v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
}

// eight numbers as they lie in memory
template <typename T> struct Eight;
template <> struct Eight<float> {
    float4 a, b;
    __device__ __forceinline__ void load(const float* p) { a = __ldcs(reinterpret_cast<const float4*>(p)); b = __ldcs(reinterpret_cast<const float4*>(p + 4)); }
    __device__ __forceinline__ void zero() { a = b = make_float4(0.f, 0.f, 0.f, 0.f); }
    __device__ __forceinline__ void get(float (&v)[8]) const { v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w; }
};
template <> struct Eight<__nv_bfloat16> {
    uint4 r;
    __device__ __forceinline__ void load(const __nv_bfloat16* p) { r = __ldcs(reinterpret_cast<const uint4*>(p)); }
    __device__ __forceinline__ void zero() { r = make_uint4(0u, 0u, 0u, 0u); }
    __device__ __forceinline__ void get(float (&v)[8]) const {
        const unsigned w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[2 * i] = __uint_as_float(w[i] << 16);
            v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        }
    }
};

// codes of the eight numbers at column d of a row and, from the first lane of a block, its scale byte; the last block of a
// row also clears the places behind it
__device__ __forceinline__ void keep8(const uint2& bytes, int e, unsigned char* codes, unsigned char* scales, int d, int K) {
    if (d < K) {
        *reinterpret_cast<uint2*>(codes + d) = bytes;
        if (d % FP8_BLOCK == 0) {
            scales[d / FP8_BLOCK] = (unsigned char)(e + 127);
            if (d + FP8_BLOCK >= K)
                for (int j = d / FP8_BLOCK + 1; j < fp8_scale_pitch(K); ++j) scales[j] = 0;
        }
    }
}
__device__ __forceinline__ void leave8(const float (&v)[8], unsigned char* codes, unsigned char* scales, int d, int K) {
    uint2 bytes;
    const int e = fp8_encode8(v, bytes);
    keep8(bytes, e, codes, scales, d, K);
}

// FORM 0: the rows; 1: act(x); 2: gated act of the row's halves (x has 2 K columns); 3: the rows, each left at `top` places
// (the rows that a token's choices of experts have in the sorted order).  grid (rows, chunks of 2,048 columns): eight columns a thread.  (Two rows a
// thread, all asked for before the first is used: 1,531 rows of gates and ups of 14,336 22.4 us by silu, 25.6 by gelu's tanh form; one 22.3 and 24.8.)
template <typename T, int FORM, int ACT>
__global__ void __launch_bounds__(ROWS_THREADS) rows_kernel(const T* __restrict__ x, unsigned char* __restrict__ codes,
                                                            unsigned char* __restrict__ scales, int K, Fp8Gate gp,
                                                            const int* __restrict__ place, int top) {
    grid_launch_dependents();
    grid_dependency_wait();
    const size_t row = blockIdx.x;
    const int d = (blockIdx.y * ROWS_THREADS + threadIdx.x) * 8, pitch = fp8_scale_pitch(K);
    constexpr int HALVES = FORM == 2 ? 2 : 1;
    Eight<T> raw[HALVES];
#pragma unroll
    for (int h = 0; h < HALVES; ++h)
        if (d < K) raw[h].load(x + (row * HALVES + h) * K + d);
        else raw[h].zero();
    float v[8];
    raw[0].get(v);
    if (FORM == 1)
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = fp8_act(v[i], ACT);
    if (FORM == 2) {
        float u[8];
        raw[HALVES - 1].get(u);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = fp8_gated(v[i], u[i], ACT, gp);
    }
    uint2 bytes;
    const int e = fp8_encode8(v, bytes);
    if (FORM == 3) {
        for (int k = 0; k < top; ++k) {
            const int to_row = place[row * top + k];
            if (to_row < 0) continue;
            const size_t to = to_row;
            keep8(bytes, e, codes + to * K, scales + to * pitch, d, K);
        }
    } else {
        keep8(bytes, e, codes + row * K, scales + row * pitch, d, K);
    }
}

// y = x * (f_hi + f_lo) * w, rounded to float32 once: t + rest_t is the row's number under the norm, u what rest_t makes of y.
struct Product { float t, u, y; };
__device__ __forceinline__ Product product_of(float x, float f_hi, float f_lo, float w) {
    const float t = x * f_hi, u = fmaf(x, f_lo, fmaf(x, f_hi, -t)) * w;
    return {t, u, fmaf(t, w, u)};
}
// Rounded twice, a number next to a border of E4M3 may land on the border and fall to the wrong side.  Borders, those of the scales among them,
// end in 19 bits of 0.  (So does one number in 2^19.)
__device__ __forceinline__ bool may_be_a_border(float y) { return (__float_as_uint(y) & 0x7ffffu) == 0u; }
// such a y, moved to its neighbour on the number's own side
__device__ __forceinline__ float beside_border(const Product& p, float w) {
    const float rest = fmaf(p.t, w, -p.y) + p.u;
    const unsigned b = __float_as_uint(p.y);
    // (a rest of less than 2^-44 is what the sums and the two halves of the factor are off by: the number itself may well stand on the border)
    if (fabsf(rest) > fabsf(p.y) * 0x1p-44f && fabsf(rest) < INFINITY && p.y != 0.f) return __uint_as_float((rest > 0.f) == (p.y > 0.f) ? b + 1u : b - 1u);
    return p.y;
}

// A CTA to a row, which stays in registers: SLOTS times eight numbers a thread.  delta: splits planes `plane` elements apart
// (partial sums, added in order), or null.  The squares are summed in 64 bits and the factor is held in two float32, so that the one
// rounding is E4M3's (in 32 bits one number in a million fell to the wrong side of a border, up to ten in 2,048 rows of 4,096; 19.3 us then,
// 20.5 so).  Registers are held to what lets as many CTAs onto an SM as before: without that 21.5.
template <typename TD, int SLOTS, int THREADS>
__global__ void __launch_bounds__(THREADS, THREADS == 1024 ? 1 : SLOTS == 1 ? 6 : SLOTS == 2 ? 5 : sizeof(TD) == 2 ? 4 : 3) norm_kernel(float* __restrict__ h, const TD* __restrict__ delta, int splits, long long plane,
                                                    const float* __restrict__ weight, unsigned char* __restrict__ codes,
                                                    unsigned char* __restrict__ scales, int K, float eps) {
    __shared__ double part[32];
    grid_launch_dependents();
    grid_dependency_wait();
    const size_t row = blockIdx.x;
    float* hr = h + row * K;
    float x[SLOTS][8];
    double ss = 0.0;
#pragma unroll
    for (int s = 0; s < SLOTS; ++s) {
        const int d = (s * blockDim.x + threadIdx.x) * 8;
        if (d < K) {
            load8(hr + d, x[s]);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) x[s][i] = 0.f;
        }
    }
    if (delta != nullptr) {
#pragma unroll
        for (int s = 0; s < SLOTS; ++s) {
            const int d = (s * blockDim.x + threadIdx.x) * 8;
            if (d < K) {
                float y[8];
                load8(delta + row * K + d, y);
                for (int sp = 1; sp < splits; ++sp) {
                    float z[8];
                    load8(delta + sp * plane + row * K + d, z);
#pragma unroll
                    for (int i = 0; i < 8; ++i) y[i] += z[i];
                }
#pragma unroll
                for (int i = 0; i < 8; ++i) x[s][i] += y[i];
                *reinterpret_cast<float4*>(hr + d) = make_float4(x[s][0], x[s][1], x[s][2], x[s][3]);
                *reinterpret_cast<float4*>(hr + d + 4) = make_float4(x[s][4], x[s][5], x[s][6], x[s][7]);
            }
        }
    }
#pragma unroll
    for (int s = 0; s < SLOTS; ++s) {
        double q[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const double lo = x[s][i], hi = x[s][i + 4];
            q[i] = fma(hi, hi, lo * lo);
        }
        ss += (q[0] + q[1]) + (q[2] + q[3]);
    }
    auto sum64 = [](double v) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
        return v;
    };
    ss = sum64(ss);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, n_warps = blockDim.x >> 5;
    if (lane == 0) part[warp] = ss;
    __syncthreads();
    const double factor = rsqrt(sum64(lane < n_warps ? part[lane] : 0.0) / K + (double)eps);
    const float f_hi = (float)factor, f_lo = (float)(factor - (double)f_hi);
#pragma unroll
    for (int s = 0; s < SLOTS; ++s) {
        const int d = (s * blockDim.x + threadIdx.x) * 8;
        if (s * (int)blockDim.x * 8 >= K) break;
        if (d < K) {
            float w[8];
            load8(weight + d, w);
            bool border = false;
#pragma unroll
            for (int i = 0; i < 8; ++i) border |= may_be_a_border(product_of(x[s][i], f_hi, f_lo, w[i]).y);
            if (border) {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const Product p = product_of(x[s][i], f_hi, f_lo, w[i]);
                    x[s][i] = may_be_a_border(p.y) ? beside_border(p, w[i]) : p.y;
                }
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) x[s][i] = product_of(x[s][i], f_hi, f_lo, w[i]).y;
            }
        }
        leave8(x[s], codes + row * K, scales + row * fp8_scale_pitch(K), d, K);
    }
}

// The (token, choice) pairs sorted by expert, stably, and the tiles of rows that the experts' products walk: one CTA.  A warp has a run of
// the pairs and counts them by expert, 32 at a time; prefix sums over the warps and over the experts say where every warp's
// pairs of an expert start; then the warps walk their runs again and place them.  (2,048 tokens of 4 choices: 34 us when a warp
// walked all pairs for each expert.)
// order[position] = pair; place[pair] = position, -1 where chosen is no expert; tiles: their number, then TILE_INTS for each: expert, first row,
// rows.  An expert's tiles are even shares of its rows, `width` rows at most.
constexpr int TILE_INTS = 3;
__global__ void __launch_bounds__(1024) plan_kernel(const int* __restrict__ chosen, int n_pairs, int n_experts, int width, int warps, int* __restrict__ order,
                                                    int* __restrict__ place, int* __restrict__ tiles, int most_tiles) {
    extern __shared__ int counts[];                   // [warps][n_experts]
    int* const first = counts + warps * n_experts;    // [n_experts]: where an expert's rows start
    int* const total = first + n_experts;             // [n_experts]
    int* const tile0 = total + n_experts;             // [n_experts]: its first tile
    grid_launch_dependents();
    grid_dependency_wait();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (int i = threadIdx.x; i < warps * n_experts; i += blockDim.x) counts[i] = 0;
    __syncthreads();
    const int per = ((n_pairs + warps - 1) / warps + 31) / 32 * 32;
    const int from = warp * per, to = min(from + per, n_pairs);
    int* const mine = counts + warp * n_experts;
    // e: the lane's expert or -1; its pairs before this one, of this warp
    auto rank_of = [&](int e) {
        const unsigned alike = __match_any_sync(0xffffffffu, e >= 0 ? e : -1);
        const int before = __popc(alike & ((1u << lane) - 1u)), base = e >= 0 ? mine[e] : 0;
        __syncwarp();
        if (e >= 0 && before == 0) mine[e] = base + __popc(alike);
        __syncwarp();
        return base + before;
    };
    auto expert_of = [&](int a) {
        const int e = a < to ? chosen[a] : -1;
        return e < n_experts ? e : -1;
    };
    if (warp < warps)
        for (int a = from; a < to; a += 32) rank_of(max(expert_of(a + lane), -1));
    __syncthreads();
    for (int e = threadIdx.x; e < n_experts; e += blockDim.x) {
        int s = 0;
        for (int w = 0; w < warps; ++w) {
            const int c = counts[w * n_experts + e];
            counts[w * n_experts + e] = s;
            s += c;
        }
        total[e] = s;
    }
    __syncthreads();
    auto share_of = [&](int rows) {
        const int n = (rows + width - 1) / width;
        return n > 0 ? ((rows + n - 1) / n + 15) / 16 * 16 : 1;
    };
    if (warp == 0) {
        int rows = 0, n = 0;
        for (int e0 = 0; e0 < n_experts; e0 += 32) {
            const int r = e0 + lane < n_experts ? total[e0 + lane] : 0, share = share_of(r), k = (r + share - 1) / share;
            int sr = r, sk = k;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int a = __shfl_up_sync(0xffffffffu, sr, o), b = __shfl_up_sync(0xffffffffu, sk, o);
                if (lane >= o) { sr += a; sk += b; }
            }
            if (e0 + lane < n_experts) {
                first[e0 + lane] = rows + sr - r;
                tile0[e0 + lane] = n + sk - k;
            }
            rows += __shfl_sync(0xffffffffu, sr, 31);
            n += __shfl_sync(0xffffffffu, sk, 31);
        }
        if (lane == 0) tiles[0] = min(n, most_tiles);
    }
    __syncthreads();
    if (warp < warps)
        for (int a = from; a < to; a += 32) {
            const int e = max(expert_of(a + lane), -1), at = rank_of(e) + (e >= 0 ? first[e] : 0);
            if (a + lane < to) {
                place[a + lane] = e >= 0 ? at : -1;
                if (e >= 0) order[at] = a + lane;
            }
        }
    for (int e = threadIdx.x; e < n_experts; e += blockDim.x) {
        const int rows = total[e], share = share_of(rows), n = (rows + share - 1) / share;
        for (int i = 0; i < n; ++i) {
            if (tile0[e] + i >= most_tiles) break;
            int* t = tiles + 1 + TILE_INTS * (tile0[e] + i);
            t[0] = e;
            t[1] = first[e] + i * share;
            t[2] = min(share, rows - i * share);
        }
    }
}

template <typename T, int FORM, int ACT>
int launch_rows_act(const void* x, void* codes, void* scales, int rows, int K, const Fp8Gate& gp, const int* place, int top, cudaStream_t s) {
    const dim3 grid(rows, (K + 8 * ROWS_THREADS - 1) / (8 * ROWS_THREADS));
    return (int)tl_launch(rows_kernel<T, FORM, ACT>, grid, dim3(ROWS_THREADS), 0, s, (const T*)x, (unsigned char*)codes, (unsigned char*)scales, K, gp, place, top);
}
template <typename T>
int launch_rows(const void* x, void* codes, void* scales, int rows, int K, int form, int act, const Fp8Gate& gp, const int* place, int top,
                cudaStream_t s) {
    if (form == 0) return launch_rows_act<T, 0, 0>(x, codes, scales, rows, K, gp, place, top, s);
    if (form == 3) return launch_rows_act<T, 3, 0>(x, codes, scales, rows, K, gp, place, top, s);
#define TL_ACT(A) return form == 1 ? launch_rows_act<T, 1, A>(x, codes, scales, rows, K, gp, place, top, s) : launch_rows_act<T, 2, A>(x, codes, scales, rows, K, gp, place, top, s)
    if (act == FP8_SILU) TL_ACT(FP8_SILU);
    if (act == FP8_GELU_TANH) TL_ACT(FP8_GELU_TANH);
    if (act == FP8_RELU2) TL_ACT(FP8_RELU2);
    if (act == FP8_GELU) TL_ACT(FP8_GELU);
#undef TL_ACT
    return launch_rows_act<T, 2, FP8_CLAMPED_SWISH>(x, codes, scales, rows, K, gp, place, top, s);
}

template <typename TD>
int launch_norm(float* h, const void* delta, int splits, long long plane, const float* weight, void* codes, void* scales, int rows, int K,
                float eps, cudaStream_t s) {
    const int lanes = (K + FP8_BLOCK - 1) / FP8_BLOCK * 16;        // whole blocks
    auto threads = [&](int slots) { return ((lanes + slots - 1) / slots + 31) / 32 * 32; };
    unsigned char *c = (unsigned char*)codes, *b = (unsigned char*)scales;
#define TL_NORM(S, T) return (int)tl_launch(norm_kernel<TD, S, T>, dim3(rows), dim3(threads(S)), 0, s, h, (const TD*)delta, splits, plane, weight, c, b, K, eps)
    // Few rows: as many threads as there are eights of numbers.  Many: small CTAs, of which more fit an SM, each somewhere else on its
    // way from loads to stores (2,048 rows of 4,096 20.5 us, with 512 threads 22.7, floor 14.1; of 2,048 10.6 and 12.2, of 8,192 41.7 and 47.3; 512
    // rows, as many threads as eights, 7.9).
    if (rows >= 4 * 148) {
        if (lanes <= 256) TL_NORM(1, 256);
        if (lanes <= 512) TL_NORM(2, 256);
        if (lanes <= 1024) TL_NORM(4, 256);
    }
    if (lanes <= 1024) TL_NORM(1, 1024);
    if (lanes <= 2048) TL_NORM(2, 1024);
    TL_NORM(4, 1024);
#undef TL_NORM
}

}  // namespace

constexpr int FP8_MOST_NORM_WIDTH = 32768;

namespace {
int rows_of(const void* x, int dtype, void* codes, void* scales, int rows, int K, int form, int act, const Fp8Gate& gp, const int* place, int top,
            cudaStream_t s) {
    if (rows <= 0) return TL_OK;
    if (K <= 0 || K % 16 != 0 || K > (1 << 26)) return TL_BAD_SIZE;
    if (!aligned16(x) || !aligned16(codes) || (reinterpret_cast<uintptr_t>(scales) & 3u) != 0) return TL_BAD_ALIGN;
    if (dtype == TL_F32) return launch_rows<float>(x, codes, scales, rows, K, form, act, gp, place, top, s);
    if (dtype == TL_BF16) return launch_rows<__nv_bfloat16>(x, codes, scales, rows, K, form, act, gp, place, top, s);
    return TL_BAD_DTYPE;
}
}  // namespace

// x: [rows, K] of dtype (form 2: [rows, 2 K]); codes [rows, K]; scales [rows, fp8_scale_pitch(K)]; all 16-byte aligned (scales: 4).
// form 0: the rows, 1: act(x), 2: act(first half) * second half; act as in fp8.cuh.
extern "C" int tl_fp8_rows(const void* x, int dtype, void* codes, void* scales, int rows, int K, int form, int act, float limit, float alpha,
                           float up_offset, void* stream) {
    if (form < 0 || form > 2 || act < 0 || act > 4 || (act == FP8_CLAMPED_SWISH && form == 1)) return TL_BAD_SIZE;
    return rows_of(x, dtype, codes, scales, rows, K, form, act, Fp8Gate{limit, alpha, up_offset}, nullptr, 1, (cudaStream_t)stream);
}

// x: [tokens, K]; codes, scales: [tokens * top] rows, token t's at place[t * top], .. place[t * top + top - 1].
extern "C" int tl_fp8_rows_placed(const void* x, int dtype, void* codes, void* scales, int tokens, int K, const int* place, int top, void* stream) {
    if (top < 1 || place == nullptr) return TL_BAD_SIZE;
    return rows_of(x, dtype, codes, scales, tokens, K, 3, 0, Fp8Gate{0.f, 0.f, 0.f}, place, top, (cudaStream_t)stream);
}

// h [rows, K] float32, updated in place when delta is not null; delta [splits, rows, K] of delta_dtype, planes `plane` elements apart.
extern "C" int tl_fp8_norm(float* h, const void* delta, int delta_dtype, int splits, long long plane, const float* weight, void* codes,
                           void* scales, int rows, int K, float eps, void* stream) {
    if (rows <= 0) return TL_OK;
    if (K <= 0 || K % 16 != 0 || K > FP8_MOST_NORM_WIDTH || splits < 1 || plane % 8 != 0) return TL_BAD_SIZE;
    if (!aligned16(h) || !aligned16(delta) || !aligned16(weight) || !aligned16(codes) || (reinterpret_cast<uintptr_t>(scales) & 3u) != 0)
        return TL_BAD_ALIGN;
    if (delta_dtype == TL_F32) return launch_norm<float>(h, delta, splits, plane, weight, codes, scales, rows, K, eps, (cudaStream_t)stream);
    if (delta_dtype == TL_BF16) return launch_norm<__nv_bfloat16>(h, delta, splits, plane, weight, codes, scales, rows, K, eps, (cudaStream_t)stream);
    return TL_BAD_DTYPE;
}

// chosen: int32 [n_pairs]; order, place: int32 [n_pairs]; tiles: int32 [1 + 3 * most_tiles] (see plan_kernel), most_tiles at least
// min(n_pairs, ceil(n_pairs / width) + n_experts).
extern "C" int tl_fp8_plan(const int* chosen, int n_pairs, int n_experts, int width, int* order, int* place, int* tiles, int most_tiles, void* stream) {
    if (n_pairs <= 0) return TL_OK;
    if (n_experts <= 0 || n_experts > 4096 || width < 16 || width % 16 != 0) return TL_BAD_SIZE;
    const long long most = ((long long)n_pairs + width - 1) / width + n_experts;
    if (most_tiles < (most < n_pairs ? most : n_pairs)) return TL_BAD_SIZE;
    const int room = 48 * 1024 / 4 / n_experts - 3;                  // rows of ints (beyond 48 KB: up to 200)
    int warps = n_pairs < 1024 ? (n_pairs + 31) / 32 : 32;
    if (warps > room) warps = room < 8 ? (warps < 8 ? warps : 8) : room;
    const size_t smem = (size_t)(warps + 3) * n_experts * sizeof(int);
    if (smem > 48 * 1024) {
        const cudaError_t e = cudaFuncSetAttribute(plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 200 * 1024);
        if (e != cudaSuccess) return (int)e;
    }
    return (int)tl_launch(plan_kernel, dim3(1), dim3(1024), smem, (cudaStream_t)stream, chosen, n_pairs, n_experts, width, warps, order, place, tiles, most_tiles);
}
