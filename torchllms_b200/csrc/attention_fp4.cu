// Attention over a paged cache of 4-bit keys and values (fp4.cuh): the kernel that takes every size.
//
//     o[t, h] = sum_j w_j v_j / sum_j w_j,   w_j = exp(scale q[t, h] . k_j)
// over the visible keys j of the token's request: j <= pos(t), and j > pos(t) - window where there is a window; pos(t) is the
// token's place in its request, kv_len - q_len + its number.  Query head h reads key head h / (H / KV).  A row that sees no key
// (a request whose length is less than its new tokens) is zeros.
//
// A CTA to a token and query head, four warps that take blocks of 32 keys in turn, each with a running maximum and sum and float32
// accumulators, joined at the end.  A lane has a key while scores are taken (its dot product is its own, no exchange) and
// coordinates while values are added up.  All arithmetic is float32 multiply-adds: a cached number times its scale is exact.
//
// It serves head sizes that the tensor-core kernels do not take (any multiple of 16 up to 256) and is bound by instruction issue:
// every query head of a group unpacks the keys and values again.  One token of 8 requests of 2,049, 32 / 8 heads: of 96 166 us, of 256 226 us; of
// 128 174 us where the tensor-core kernel takes 11.9.
#include "fp4.cuh"
#include <math.h>

namespace {

constexpr int WARPS = 4;
constexpr int MAX_DIM = 256;
constexpr float LOG2E = 1.4426950408889634f;

struct GeneralParams {
    const unsigned char* k_pages;
    const unsigned char* v_pages;
    const int* block_table;
    const int* q_start;
    const int* kv_len;
    long long n_pages;
    int table_stride, table_cols;
    int n_heads, n_kv_heads, head_dim, page_size, window;
    float scale_log2;
};

template <typename T>
__global__ void __launch_bounds__(WARPS * 32) attention_fp4_general_kernel(const T* __restrict__ q, T* __restrict__ out, const GeneralParams p) {
    __shared__ float qs[MAX_DIM];
    __shared__ float acc_s[WARPS][MAX_DIM];
    __shared__ float m_s[WARPS], l_s[WARPS];
    grid_launch_dependents();
    grid_dependency_wait();
    const int b = blockIdx.z, h = blockIdx.y, D = p.head_dim;
    const int first = p.q_start[b], ql = p.q_start[b + 1] - first;
    if ((int)blockIdx.x >= ql) return;
    const int pos = p.kv_len[b] - ql + (int)blockIdx.x;
    const size_t row = ((size_t)(first + blockIdx.x) * p.n_heads + h) * D;
    const int kvh = h / (p.n_heads / p.n_kv_heads);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (int d = threadIdx.x; d < D; d += blockDim.x) qs[d] = to_float(q[row + d]);
    __syncthreads();

    const int lo = p.window > 0 ? max(0, pos - p.window + 1) : 0;
    const int hi = min(pos + 1, p.table_cols * p.page_size);           // keys lo .. hi - 1
    const int* table = p.block_table + (size_t)b * p.table_stride;
    float m = -INFINITY, l = 0.f;
    float acc[MAX_DIM / 64][2];
#pragma unroll
    for (int i = 0; i < MAX_DIM / 64; ++i) acc[i][0] = acc[i][1] = 0.f;
    for (int k0 = (lo & ~31) + warp * 32; k0 < hi; k0 += WARPS * 32) {
        const int kpos = k0 + lane;
        const bool visible = kpos >= lo && kpos < hi;
        Fp4Place at = {0, 0};
        float s = -INFINITY;
        if (visible) {
            long long page = table[kpos / p.page_size];
            if (!tl_check_page(page) || page < 0 || page >= p.n_pages) page = 0;      // (a bad page is not followed; debug builds report it)
            at = fp4_place(page, kpos % p.page_size, kvh, p.n_kv_heads, p.page_size, D);
            float dot = 0.f;
            for (int g = 0; g < D / FP4_GROUP; ++g) {
                const uint2 w = *reinterpret_cast<const uint2*>(p.k_pages + at.codes + g * 8);
                __half2 r[8];
                fp4_unpack(w.x, *reinterpret_cast<__half2(*)[4]>(&r[0]));
                fp4_unpack(w.y, *reinterpret_cast<__half2(*)[4]>(&r[4]));
                float part = 0.f;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float2 v = __half22float2(r[i]);
                    part = fmaf(qs[g * FP4_GROUP + 2 * i], v.x, part);
                    part = fmaf(qs[g * FP4_GROUP + 2 * i + 1], v.y, part);
                }
                dot = fmaf(part, fp4_scale(p.k_pages[at.scales + g]), dot);
            }
            s = dot * p.scale_log2;
        }
        float top = s;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            const float other = __shfl_xor_sync(0xffffffffu, top, o);
            top = (top != top || other != other) ? NAN : fmaxf(top, other);      // (a key that is not a number shows in the result)
        }
        const float m_new = top != top ? top : fmaxf(m, top);
        const float safe = m_new == -INFINITY ? 0.f : m_new;
        const float w = visible ? exp2f(s - safe) : 0.f, shrink = exp2f(m - safe);
        m = m_new;
        l = l * shrink + w;                                             // (this lane's keys; added over the lanes at the end)
#pragma unroll
        for (int i = 0; i < MAX_DIM / 64; ++i) {
            acc[i][0] *= shrink;
            acc[i][1] *= shrink;
        }
        const unsigned seen = __ballot_sync(0xffffffffu, visible);
        for (int j = 0; j < 32; ++j) {
            if (!((seen >> j) & 1u)) continue;                          // (what lies there is not read)
            const float wj = __shfl_sync(0xffffffffu, w, j);
            const long long codes = __shfl_sync(0xffffffffu, at.codes, j), scales = __shfl_sync(0xffffffffu, at.scales, j);
#pragma unroll
            for (int i = 0; i < MAX_DIM / 64; ++i) {
                const int d2 = lane + 32 * i;                           // the byte, with coordinates 2 d2 and 2 d2 + 1
                if (d2 < D / 2) {
                    const __half2 r = fp4_unpack2(p.v_pages[codes + d2]);
                    const float2 v = __half22float2(__hmul2(r, fp4_scale2(p.v_pages[scales + d2 / (FP4_GROUP / 2)])));
                    acc[i][0] = fmaf(wj, v.x, acc[i][0]);
                    acc[i][1] = fmaf(wj, v.y, acc[i][1]);
                }
            }
        }
    }
    l = warp_sum(l);
    if (lane == 0) {
        m_s[warp] = m;
        l_s[warp] = l;
    }
#pragma unroll
    for (int i = 0; i < MAX_DIM / 64; ++i)
        if (lane + 32 * i < D / 2) {
            acc_s[warp][2 * (lane + 32 * i)] = acc[i][0];
            acc_s[warp][2 * (lane + 32 * i) + 1] = acc[i][1];
        }
    __syncthreads();
    float M = -INFINITY;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) M = (M != M || m_s[w] != m_s[w]) ? NAN : fmaxf(M, m_s[w]);
    float den = 0.f, f[WARPS];
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
        f[w] = m_s[w] == -INFINITY ? 0.f : exp2f(m_s[w] - M);
        den = fmaf(f[w], l_s[w], den);
    }
    // (no sum: zeros for a row without a key; where all scores are -inf, from a query that is not finite, there is no softmax)
    const float inv = M == -INFINITY ? (pos >= 0 ? NAN : 0.f) : 1.f / den;
    for (int d = threadIdx.x; d < D; d += blockDim.x) {
        float num = 0.f;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) num = fmaf(f[w], acc_s[w][d], num);
        out[row + d] = from_float<T>(num * inv);
    }
}

}  // namespace

// q, out: [tokens, n_heads, head_dim] of dtype; pages: [n_pages, n_kv_heads, page_size / 16, 9 head_dim] bytes.  q_start may count from
// anywhere in q; block_table: [n_seqs, table_cols] with rows table_stride apart.
extern "C" int tl_attention_fp4_general(const void* q, const void* k_pages, const void* v_pages, void* out, const int* block_table,
                                        int table_stride, int table_cols, const int* q_start, const int* kv_len, int dtype, int n_seqs,
                                        int n_heads, int n_kv_heads, int head_dim, int page_size, long long n_pages, int max_q_len,
                                        int window, float scale, void* stream) {
    if (n_seqs <= 0 || max_q_len <= 0) return TL_OK;
    if (n_heads <= 0 || n_kv_heads <= 0 || n_heads % n_kv_heads != 0 || n_heads > 65535 || n_seqs > 65535 || n_pages <= 0) return TL_BAD_SIZE;
    if (head_dim < FP4_GROUP || head_dim > MAX_DIM || head_dim % FP4_GROUP != 0 || page_size < FP4_RECORD || page_size % FP4_RECORD != 0)
        return TL_BAD_SIZE;
    if (!fp4_places_fit(table_cols, page_size, max_q_len)) return TL_BAD_SIZE;
    if (!aligned16(k_pages) || !aligned16(v_pages)) return TL_BAD_ALIGN;
    const GeneralParams p = {(const unsigned char*)k_pages, (const unsigned char*)v_pages, block_table, q_start, kv_len, n_pages, table_stride,
                             table_cols, n_heads, n_kv_heads, head_dim, page_size, fp4_window(window, table_cols, page_size), scale * LOG2E};
    const dim3 grid((unsigned)max_q_len, (unsigned)n_heads, (unsigned)n_seqs);
    cudaStream_t s = (cudaStream_t)stream;
    if (dtype == TL_BF16)
        return (int)tl_launch(attention_fp4_general_kernel<__nv_bfloat16>, grid, dim3(WARPS * 32), 0, s, (const __nv_bfloat16*)q, (__nv_bfloat16*)out, p);
    if (dtype == TL_F32)
        return (int)tl_launch(attention_fp4_general_kernel<float>, grid, dim3(WARPS * 32), 0, s, (const float*)q, (float*)out, p);
    return TL_BAD_DTYPE;
}
