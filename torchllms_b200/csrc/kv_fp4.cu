// Writing a paged cache of 4-bit keys and values with the rotation on the way, and reading it back.
//
// rope_kv_write_fp4: a token's projected row is [q heads | k heads | v heads].  The first rot_dims coordinates of every q and
// k head are rotated by the angles of the token's position, pairs (2i, 2i + 1) or (i, i + rot_dims / 2):
//     y0 = x0 cos - x1 sin,  y1 = x1 cos + x0 sin
// in float32, every product and sum rounded by itself (no fused multiply-add: what goes into the cache is then the same
// number whichever kernel or program rotates, and a code does not flip).  q leaves rounded once; k and v are not
// rounded before they become 4-bit numbers (fp4.cuh), which happens in the same registers: a thread has eight coordinates, a
// pair of lanes the sixteen of a group.
//
// Bound by memory: a row is read once, q and 4.5 bits a number of k and v are written.
#include "fp4.cuh"

namespace {

// eight consecutive elements as floats
__device__ __forceinline__ void load8(const float* p, float (&x)[8]) {
    const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
    x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w; x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
}
__device__ __forceinline__ void load8(const __nv_bfloat16* p, float (&x)[8]) {
    Vec16<__nv_bfloat16> v;
    v.load(p);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = v.get(i);
}
__device__ __forceinline__ void store8(float* p, const float (&x)[8]) {
    *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]);
    *reinterpret_cast<float4*>(p + 4) = make_float4(x[4], x[5], x[6], x[7]);
}
__device__ __forceinline__ void store8(__nv_bfloat16* p, const float (&x)[8]) {
    Vec16<__nv_bfloat16> v;
#pragma unroll
    for (int i = 0; i < 8; ++i) v.set(i, x[i]);
    v.store(p);
}

struct WriteParams {
    const int* positions;
    const float* table;            // [table_rows, rot_dims / 2, 2]
    const int* slot_mapping;
    unsigned char* k_pages;
    unsigned char* v_pages;
    long long plane, n_pages;
    int splits, n_tokens, n_heads, n_kv_heads, head_dim, rot_dims, page_size, table_rows;
    RowScale rs;
};

// eight coordinates of a row, its planes added up and scaled
template <typename TI>
__device__ __forceinline__ void fetch8(const TI* src, const WriteParams& p, float sc, float (&x)[8]) {
    load8(src, x);
    for (int sp = 1; sp < p.splits; ++sp) {
        float y[8];
        load8(src + sp * p.plane, y);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] += y[i];
    }
    if (p.rs.ssq != nullptr) {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] *= sc;
    }
}
template <typename TI>
__device__ __forceinline__ float fetch1(const TI* src, const WriteParams& p, float sc) {
    float x = to_float(*src);
    for (int sp = 1; sp < p.splits; ++sp) x += to_float(src[sp * p.plane]);
    return p.rs.ssq != nullptr ? x * sc : x;
}

// A CTA (or several, blockIdx.y) to a token, a thread to a run of eight coordinates at a time; a head has an even number of
// runs and a CTA an even number of threads, so the two runs of a group are neighbouring lanes.  A decoded token of 48 heads of 64: 2.2 us, a launch
// and its latency; 64 tokens of 48 heads of 128 2.7.
template <typename TI, typename T, bool INTERLEAVED>
__global__ void __launch_bounds__(128) rope_kv_write_fp4_kernel(const TI* __restrict__ qkv, T* __restrict__ q_out, const WriteParams p) {
    grid_launch_dependents();
    grid_dependency_wait();
    const int t = blockIdx.x;
    const float sc = warp_row_scale(p.rs, t);
    const int per_head = p.head_dim >> 3, heads = p.n_heads + 2 * p.n_kv_heads, runs = heads * per_head;
    int pos = p.positions[t];
    (void)TL_CHECK(pos >= 0 && pos < p.table_rows, TL_DBG_POSITION);
    pos = pos < 0 ? 0 : (pos >= p.table_rows ? p.table_rows - 1 : pos);   // the host keeps positions inside the table
    const float* cs = p.table + (size_t)pos * p.rot_dims;
    const TI* src = qkv + (size_t)t * heads * p.head_dim;
    long long page = 0;
    int slot = 0;
    bool write = p.k_pages != nullptr;
    if (write) {
        const int sm = p.slot_mapping[t];
        page = sm / p.page_size;
        slot = sm - (int)page * p.page_size;
        // (a slot outside the cache is not written; debug builds report it)
        write = TL_CHECK(sm >= 0, TL_DBG_SLOT) && tl_check_page(page) && sm >= 0 && page < p.n_pages;
    }
    const int half = p.rot_dims >> 1;
    // (whole warps go round together: the lanes of a group exchange their maxima)
    for (int c0 = blockIdx.y * blockDim.x; c0 < runs; c0 += gridDim.y * blockDim.x) {
        const int c = c0 + threadIdx.x;
        const bool mine = c < runs;
        const int head = mine ? c / per_head : 0;
        const int off = mine ? (c - head * per_head) << 3 : 0;
        float x[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = 0.f;
        if (mine) {
            fetch8(src + head * p.head_dim + off, p, sc, x);
            if (head < p.n_heads + p.n_kv_heads && off < p.rot_dims) {
                if (INTERLEAVED) {
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (off + 2 * i < p.rot_dims) {
                            const float2 r = *reinterpret_cast<const float2*>(cs + off + 2 * i);
                            const float a = x[2 * i], b = x[2 * i + 1];
                            x[2 * i] = __fsub_rn(__fmul_rn(a, r.x), __fmul_rn(b, r.y));
                            x[2 * i + 1] = __fadd_rn(__fmul_rn(b, r.x), __fmul_rn(a, r.y));
                        }
                } else if ((half & 7) == 0) {
                    // the partners are another whole run
                    const bool first = off < half;
                    float y[8];
                    fetch8(src + head * p.head_dim + (first ? off + half : off - half), p, sc, y);
                    const float* r = cs + 2 * (first ? off : off - half);
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const float2 a = *reinterpret_cast<const float2*>(r + 2 * i);
                        const float u = __fmul_rn(x[i], a.x), v = __fmul_rn(y[i], a.y);
                        x[i] = first ? __fsub_rn(u, v) : __fadd_rn(u, v);
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const int d = off + i;
                        if (d < p.rot_dims) {
                            const bool first = d < half;
                            const float y = fetch1(src + head * p.head_dim + (first ? d + half : d - half), p, sc);
                            const float2 a = *reinterpret_cast<const float2*>(cs + 2 * (first ? d : d - half));
                            const float u = __fmul_rn(x[i], a.x), v = __fmul_rn(y, a.y);
                            x[i] = first ? __fsub_rn(u, v) : __fadd_rn(u, v);
                        }
                    }
                }
            }
        }
        unsigned top = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(x[i]) & 0x7fffffffu);
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
        if (!mine) continue;
        if (head < p.n_heads) {
            store8(q_out + ((size_t)t * p.n_heads + head) * p.head_dim + off, x);
        } else if (write) {
            const bool is_k = head < p.n_heads + p.n_kv_heads;
            const int kvh = is_k ? head - p.n_heads : head - p.n_heads - p.n_kv_heads;
            unsigned char* base = is_k ? p.k_pages : p.v_pages;
            const Fp4Place at = fp4_place(page, slot, kvh, p.n_kv_heads, p.page_size, p.head_dim);
            const unsigned byte = fp4_scale_byte(top);
            *reinterpret_cast<unsigned*>(base + at.codes + off / 2) = fp4_pack8(x, byte);
            if ((off & 8) == 0) base[at.scales + off / FP4_GROUP] = (unsigned char)byte;
        }
    }
}

// The same for rows of one plane and of the type that q leaves in, heads of a power of two up to 1,024 and many tokens: a thread's runs lie a
// multiple of the head size apart, so that one run of the rotation table serves them all, heads come by a shift, and a
// token's loads (EACH a thread) are under way together.  Where pairs are halves a thread takes both: a run and the run of its partners
// (of what is not turned, a run of its first and one of its second half), a multiple of 16 apart.
//   8,276 tokens, 48 heads of 128, bfloat16 (179 MB, 27 us of them): 36.7 us (4.9 TB/s); with three runs at a time 40, with the kernel above
//   and divisions 72.  Without the 4-bit numbers' arithmetic it would take 32: what bounds it next to memory.  CTAs an SM, 8,276 / 4,000 / 600 tokens:
//   8 (spills) 36.4 / 17.8 / 6.0, 7 36.7 / 17.1 / 5.4, 6 38.8 / 17.6 / 4.9.
//   Halves, 4,000 tokens, float32 (168 MB, 26 us): 32.4 us (5.2 TB/s), bfloat16 20.5 (4.2 TB/s); fetching the partners beside every run 43.0 and 27.3.
template <typename T, bool INTERLEAVED> struct Runs {
    static constexpr int EACH = sizeof(T) == 2 && INTERLEAVED ? 6 : 3, PER = INTERLEAVED ? 1 : 2;
    static constexpr int CTAS = sizeof(T) == 2 ? (INTERLEAVED ? 7 : 5) : (INTERLEAVED ? 5 : 4);       // of an SM, at least: what its registers are cut to
};
template <typename T> struct Run8 {                     // eight numbers as they are stored
    uint4 v[sizeof(T) / 2];
    __device__ __forceinline__ void load(const T* p) {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i) v[i] = reinterpret_cast<const uint4*>(p)[i];
    }
    __device__ __forceinline__ float get(int i) const { return to_float(reinterpret_cast<const T*>(v)[i]); }
};
template <typename T, bool INTERLEAVED>
__global__ void __launch_bounds__(128, Runs<T, INTERLEAVED>::CTAS) rope_kv_write_fp4_rows_kernel(const T* __restrict__ qkv, T* __restrict__ q_out,
                                                                                              const int log_runs, const WriteParams p) {
    constexpr int EACH = Runs<T, INTERLEAVED>::EACH, PER = Runs<T, INTERLEAVED>::PER;      // a thread's turns at a time, runs of a turn
    grid_launch_dependents();
    grid_dependency_wait();
    const int t = blockIdx.x;
    const int log_head = log_runs + 3, log_turns = log_runs - (PER - 1);
    const int heads = p.n_heads + 2 * p.n_kv_heads, turns_all = heads << log_turns;
    const int turn = threadIdx.x & ((1 << log_turns) - 1), turned = p.rot_dims / (8 * PER);
    const bool turns = turn < turned;
    const int off = PER == 1 || turns ? turn * 8 : p.rot_dims + (turn - turned) * 8;
    const int apart = PER == 1 ? 0 : (turns ? p.rot_dims : p.head_dim - p.rot_dims) >> 1;
    // (whole runs follow one another: a turn's numbers, where it is one run, begin at 8 c)
    const T* src = qkv + (size_t)t * (heads << log_head);
    auto place = [&](int c) { return PER == 1 ? (size_t)c * 8 : ((size_t)(c >> log_turns) << log_head) + off; };
    Run8<T> raw[EACH][PER];
    auto fetch = [&](int c0) {
#pragma unroll
        for (int e = 0; e < EACH; ++e) {
            const int c = c0 + e * 128;
            if (c < turns_all) {
#pragma unroll
                for (int i = 0; i < PER; ++i) raw[e][i].load(src + place(c) + i * apart);
            }
        }
    };
    fetch(threadIdx.x);
    int pos = p.positions[t];
    (void)TL_CHECK(pos >= 0 && pos < p.table_rows, TL_DBG_POSITION);
    pos = pos < 0 ? 0 : (pos >= p.table_rows ? p.table_rows - 1 : pos);   // the host keeps positions inside the table
    long long page = 0;
    int slot = 0;
    bool write = p.k_pages != nullptr;
    if (write) {
        const int sm = p.slot_mapping[t];
        page = sm / p.page_size;
        slot = sm - (int)page * p.page_size;
        // (a slot outside the cache is not written; debug builds report it)
        write = TL_CHECK(sm >= 0, TL_DBG_SLOT) && tl_check_page(page) && sm >= 0 && page < p.n_pages;
    }
    float cs[8 * PER];
    if (turns) {
        const float* at = p.table + (size_t)pos * p.rot_dims + off * PER;
#pragma unroll
        for (int i = 0; i < 2 * PER; ++i) {
            const float4 v = *reinterpret_cast<const float4*>(at + 4 * i);
            cs[4 * i] = v.x; cs[4 * i + 1] = v.y; cs[4 * i + 2] = v.z; cs[4 * i + 3] = v.w;
        }
    }
    const float sc = warp_row_scale(p.rs, t);
    // (whole warps go round together: the lanes of a group exchange their maxima)
    for (int c0 = threadIdx.x; c0 - (int)threadIdx.x < turns_all; c0 += EACH * 128) {
        if (c0 != (int)threadIdx.x) fetch(c0);
#pragma unroll
        for (int e = 0; e < EACH; ++e) {
            const int c = c0 + e * 128;
            if (c - (int)threadIdx.x >= turns_all) break;
            const bool mine = c < turns_all;
            const int head = c >> log_turns;
            float x[PER][8];
#pragma unroll
            for (int k = 0; k < PER; ++k)
#pragma unroll
                for (int i = 0; i < 8; ++i) x[k][i] = mine ? raw[e][k].get(i) : 0.f;
            if (p.rs.ssq != nullptr) {
#pragma unroll
                for (int k = 0; k < PER; ++k)
#pragma unroll
                    for (int i = 0; i < 8; ++i) x[k][i] *= sc;
            }
            if (turns && mine && head < p.n_heads + p.n_kv_heads) {
#pragma unroll
                for (int i = 0; i < 4 * PER; ++i) {
                    float& u = PER == 1 ? x[0][2 * i] : x[0][i];
                    float& v = PER == 1 ? x[0][2 * i + 1] : x[PER - 1][i];
                    const float a = u, b = v;
                    u = __fsub_rn(__fmul_rn(a, cs[2 * i]), __fmul_rn(b, cs[2 * i + 1]));
                    v = __fadd_rn(__fmul_rn(b, cs[2 * i]), __fmul_rn(a, cs[2 * i + 1]));
                }
            }
            if (c - (int)threadIdx.x + 127 < (p.n_heads << log_turns)) {                // (the whole CTA has heads of q)
#pragma unroll
                for (int k = 0; k < PER; ++k) store8(q_out + ((size_t)t * p.n_heads << log_head) + place(c) + k * apart, x[k]);
                continue;
            }
#pragma unroll
            for (int k = 0; k < PER; ++k) {
                unsigned top = 0;
#pragma unroll
                for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(x[k][i]) & 0x7fffffffu);
                top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
                if (!mine) continue;
                if (head < p.n_heads) {
                    store8(q_out + ((size_t)t * p.n_heads << log_head) + place(c) + k * apart, x[k]);
                } else if (write) {
                    const bool is_k = head < p.n_heads + p.n_kv_heads;
                    const int kvh = is_k ? head - p.n_heads : head - p.n_heads - p.n_kv_heads, d = off + k * apart;
                    unsigned char* base = is_k ? p.k_pages : p.v_pages;
                    const Fp4Place at = fp4_place(page, slot, kvh, p.n_kv_heads, p.page_size, p.head_dim);
                    const unsigned byte = fp4_scale_byte(top);
                    *reinterpret_cast<unsigned*>(base + at.codes + d / 2) = fp4_pack8(x[k], byte);
                    if ((d & 8) == 0) base[at.scales + d / FP4_GROUP] = (unsigned char)byte;
                }
            }
        }
    }
}

// The numbers of given slots: a CTA to a slot at a time, blockIdx.y: keys, values; a thread to eight coordinates of a head, four slots
// under way together.  8,356 slots of 8 heads of 128 in bfloat16 (44 MB, 6.7 us of them): 8.6 us (5.1 TB/s; with the place of every slot and run worked out anew, a
// division and 64-bit products, 11.2), 17 slots 2.0 (2.6); eight slots at a time 11.5 and 3.4.
// (The pages are not declared free of aliases: a CTA may be resident while the kernel before this one writes them, and loads that count
// on memory nobody writes are not for them.)
constexpr int SLOTS = 4;
template <typename T>
__global__ void __launch_bounds__(128) kv_read_fp4_kernel(const unsigned char* k_pages, const unsigned char* v_pages,
                                                          const int* __restrict__ slots, T* k_out, T* v_out,
                                                          int n_slots, long long n_pages, int n_kv_heads, int head_dim, int page_size, int page_shift) {
    grid_launch_dependents();
    grid_dependency_wait();
    const unsigned char* pages = blockIdx.y ? v_pages : k_pages;
    T* out = blockIdx.y ? v_out : k_out;
    const int per_head = head_dim >> 3, runs = n_kv_heads * per_head;
    const int record = fp4_record_bytes(head_dim);
    const long long head_bytes = (long long)(page_size / FP4_RECORD) * record, page_bytes = n_kv_heads * head_bytes;
    for (int c = threadIdx.x; c < runs; c += blockDim.x) {
        const int head = c / per_head, off = (c - head * per_head) << 3;
        // where this run lies in the first slot of a page: its numbers, and its scale
        const unsigned char* numbers = pages + head * head_bytes + off / 2;
        const unsigned char* scales = pages + head * head_bytes + FP4_RECORD * (head_dim / 2) + off / FP4_GROUP;
        for (long long n0 = (long long)blockIdx.x * SLOTS; n0 < n_slots; n0 += (long long)gridDim.x * SLOTS) {
            unsigned w[SLOTS], byte[SLOTS];
#pragma unroll
            for (int i = 0; i < SLOTS; ++i) {
                w[i] = byte[i] = 0u;                    // (a slot outside the cache reads as zeros; debug builds report it)
                if (n0 + i >= n_slots) continue;
                const int sm = slots[n0 + i];
                const int page = page_shift >= 0 ? sm >> page_shift : sm / page_size;
                if (TL_CHECK(sm >= 0, TL_DBG_SLOT) && tl_check_page(page) && sm >= 0 && page < n_pages) {
                    const int slot = sm - page * page_size, row = slot & (FP4_RECORD - 1);
                    const long long at = page * page_bytes + (long long)(slot / FP4_RECORD) * record;
                    w[i] = *reinterpret_cast<const unsigned*>(numbers + at + row * (head_dim / 2));
                    byte[i] = scales[at + row * (head_dim / FP4_GROUP)];
                }
            }
            T* to = out + ((size_t)n0 * runs + c) * 8;
#pragma unroll
            for (int i = 0; i < SLOTS; ++i) {
                if (n0 + i >= n_slots) continue;
                __half2 r[4];
                fp4_unpack(w[i], r);
                const __half2 s = fp4_scale2(byte[i]);
                float x[8];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float2 v = __half22float2(__hmul2(r[e], s));      // exact
                    x[2 * e] = v.x;
                    x[2 * e + 1] = v.y;
                }
                store8(to + (size_t)i * runs * 8, x);
            }
        }
    }
}

// log2 of a power of two, or -1
int log2_of(int n) {
    for (int b = 0; b < 31; ++b)
        if (n == 1 << b) return b;
    return -1;
}

bool takes(int n_kv_heads, int head_dim, int page_size) {
    return n_kv_heads > 0 && head_dim >= FP4_GROUP && head_dim % FP4_GROUP == 0 && page_size >= FP4_RECORD && page_size % FP4_RECORD == 0;
}

}  // namespace

// qkv: [splits, n_tokens, (n_heads + 2 n_kv_heads) head_dim] of in_dtype (splits > 1 only for float32 partial sums, `plane`
// elements apart); q_out: [n_tokens, n_heads, head_dim] of dtype.  k_pages / v_pages may both be null: then only q is produced.
// in_ssq may be null; else [n_tokens, in_parts] floats give every token's row scale (RowScale in common.cuh).
extern "C" int tl_rope_kv_write_fp4(const void* qkv, int in_dtype, int splits, const int* positions, const float* table,
                                    const int* slot_mapping, void* q_out, void* k_pages, void* v_pages, int dtype, int n_tokens,
                                    int n_heads, int n_kv_heads, int head_dim, int rot_dims, int page_size, long long n_pages,
                                    int table_rows, int interleaved, const float* in_ssq, int in_parts, float in_inv_dim, float in_eps,
                                    void* stream) {
    if (n_tokens <= 0) return TL_OK;
    if (!takes(n_kv_heads, head_dim, page_size) || n_heads <= 0 || splits < 1 || table_rows <= 0) return TL_BAD_SIZE;
    if (rot_dims < 2 || rot_dims > head_dim || (rot_dims & 1)) return TL_BAD_SIZE;
    if ((k_pages == nullptr) != (v_pages == nullptr) || (in_ssq != nullptr && in_parts < 1)) return TL_BAD_SIZE;
    if (!aligned16(qkv) || !aligned16(q_out) || !aligned16(table) || !aligned16(k_pages) || !aligned16(v_pages)) return TL_BAD_ALIGN;
    WriteParams p;
    p.positions = positions; p.table = table; p.slot_mapping = slot_mapping;
    p.k_pages = (unsigned char*)k_pages; p.v_pages = (unsigned char*)v_pages;
    const int heads = n_heads + 2 * n_kv_heads;
    p.plane = (long long)n_tokens * heads * head_dim;
    p.n_pages = n_pages; p.splits = splits; p.n_tokens = n_tokens; p.n_heads = n_heads; p.n_kv_heads = n_kv_heads;
    p.head_dim = head_dim; p.rot_dims = rot_dims; p.page_size = page_size; p.table_rows = table_rows;
    p.rs = {in_ssq, in_parts, in_inv_dim, in_eps};
    const int runs = heads * (head_dim / 8);
    const int by = n_tokens >= 256 ? 1 : (runs + 127) / 128;
    cudaStream_t s = (cudaStream_t)stream;
    const int head_runs = head_dim / 8;
    if (in_dtype == dtype && splits == 1 && n_tokens >= 148 && head_runs <= 128 && (head_runs & (head_runs - 1)) == 0 &&
        rot_dims % (interleaved ? 8 : 32) == 0 && (interleaved || head_dim >= 32)) {
        int log_runs = 0;
        while ((1 << log_runs) < head_runs) ++log_runs;
#define TL_WRITE_ROWS(T, I) tl_launch(rope_kv_write_fp4_rows_kernel<T, I>, dim3(n_tokens), dim3(128), 0, s, (const T*)qkv, (T*)q_out, log_runs, p)
        if (dtype == TL_BF16) return (int)(interleaved ? TL_WRITE_ROWS(__nv_bfloat16, true) : TL_WRITE_ROWS(__nv_bfloat16, false));
        if (dtype == TL_F32) return (int)(interleaved ? TL_WRITE_ROWS(float, true) : TL_WRITE_ROWS(float, false));
#undef TL_WRITE_ROWS
    }
#define TL_WRITE(TI, T)                                                                                                         \
    (interleaved ? tl_launch(rope_kv_write_fp4_kernel<TI, T, true>, dim3(n_tokens, by), dim3(128), 0, s, (const TI*)qkv, (T*)q_out, p) \
                 : tl_launch(rope_kv_write_fp4_kernel<TI, T, false>, dim3(n_tokens, by), dim3(128), 0, s, (const TI*)qkv, (T*)q_out, p))
    if (in_dtype == TL_F32 && dtype == TL_F32) return (int)TL_WRITE(float, float);
    if (in_dtype == TL_BF16 && dtype == TL_BF16 && splits == 1) return (int)TL_WRITE(__nv_bfloat16, __nv_bfloat16);
    if (in_dtype == TL_F32 && dtype == TL_BF16) return (int)TL_WRITE(float, __nv_bfloat16);
#undef TL_WRITE
    return TL_BAD_DTYPE;
}

// k_out, v_out: [n_slots, n_kv_heads, head_dim] of dtype.
extern "C" int tl_kv_read_fp4(const void* k_pages, const void* v_pages, const int* slots, void* k_out, void* v_out, int dtype,
                              int n_slots, long long n_pages, int n_kv_heads, int head_dim, int page_size, void* stream) {
    if (n_slots <= 0) return TL_OK;
    if (!takes(n_kv_heads, head_dim, page_size)) return TL_BAD_SIZE;
    if (!aligned16(k_pages) || !aligned16(v_pages) || !aligned16(k_out) || !aligned16(v_out)) return TL_BAD_ALIGN;
    const long long groups = ((long long)n_slots + SLOTS - 1) / SLOTS;
    const unsigned bx = (unsigned)(groups < 148 * 16 ? groups : 148 * 16);
    cudaStream_t s = (cudaStream_t)stream;
    const unsigned char *k = (const unsigned char*)k_pages, *v = (const unsigned char*)v_pages;
    if (dtype == TL_BF16)
        return (int)tl_launch(kv_read_fp4_kernel<__nv_bfloat16>, dim3(bx, 2), dim3(128), 0, s, k, v, slots, (__nv_bfloat16*)k_out,
                              (__nv_bfloat16*)v_out, n_slots, n_pages, n_kv_heads, head_dim, page_size, log2_of(page_size));
    if (dtype == TL_F32)
        return (int)tl_launch(kv_read_fp4_kernel<float>, dim3(bx, 2), dim3(128), 0, s, k, v, slots, (float*)k_out, (float*)v_out, n_slots,
                              n_pages, n_kv_heads, head_dim, page_size, log2_of(page_size));
    return TL_BAD_DTYPE;
}
