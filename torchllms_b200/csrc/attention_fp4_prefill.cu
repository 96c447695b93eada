// Attention over a paged cache of 4-bit keys and values (fp4.cuh) on the fifth-generation tensor cores (head_dim 64 or 128,
// bfloat16): steps whose requests bring many tokens.
//
//     o[t, h] = sum_j w_j v_j / sum_j w_j,  w_j = exp(scale q[t, h] . k_j),  j <= pos(t), j > pos(t) - window
//
// Bound by arithmetic (4 head_dim operations a visible pair on the tensor cores, and one exponential).  The rows of a request and
// key head are (token, query head of the group): a tile of 128 rows holds 128 / group tokens with all their heads, so that keys
// and values are unpacked once for the whole group, and a tile of few tokens sees few keys that its rows do not.  A CTA
// takes two such tiles and walks the visible keys in tiles of 128; both share what is unpacked.  512 threads:
//   warps 0-3, 4-7 : softmax of row tile 0, of row tile 1, a thread to a row.  At the start they bring the rows of q to float16 (by
//                    a power of two a row that puts its largest number just below 2^15; nothing is rounded but numbers 2^-31 of
//                    the largest) into shared memory in the operand layout.  Per key tile a thread reads its 128 scores, takes the
//                    maximum, rescales the row's accumulator in the rare case that the maximum in use lags by more than 2^LAG,
//                    and writes the weights into tensor memory; at the end it divides by their sum and stores the row.
//   warps 8-11     : unpack.  A thread has a key of the tile: it converts the key's 72 bytes, fetched while it did what came before, to
//                    float16 (exact: fp4.cuh) and writes them where the products read them (128-byte-swizzled rows), then
//                    does the same with the value.
//   warp 12        : issues the scores of both row tiles, warp 13 their products with V (one elected lane each).
// Weights are multiplied as one float16 (2^-12; the result's own rounding is 2^-9), 2^BIAS times as large as they are, so that
// weights down to 2^-32 of the largest count; the row's sum carries the same factor.
//
// Scores, weights and accumulators have tensor memory of their own; the row tiles use one score buffer in turn.  Where rows are few and keys are many the keys are cut into pieces, which leave
// float32 sums that a second kernel adds up in order.
//
// Measured (32 / 8 heads, us): heads of 128: a prompt of 2,048 tokens 47.0 (730 TFLOP/s; some 6 us a CTA before its first and after its last key tile, 256
// CTAs on 148 SMs), 2,048 tokens behind 14,001 480 to 490 in a long loop (1,050 TFLOP/s, at the power cap's clock); heads of 64: six portions of 70 to
// 1,063 tokens 89 (460 TFLOP/s).  128 keys of both row tiles take 3,800 cycles with heads of 128, where the products want 2,100 and the exponentials 2,050, and 3,150
// with 64.  In copies with work taken out (of a kernel with a body for keys and one for values, 3,640 and 3,080): without the softmax 3,500 (128), without
// unpacking 2,840, without exponentials 2,280 (64): the three wait for one another.
// Measured and left out: exponentials by a polynomial on the multiply-add pipes for an eighth to a half of the scores (47 to 57 for 45.8), weights against the
// maximum in use while the new one is found (46.5; 464 for 431), a row tile held back at the start (47.3), records fetched a tile further ahead (47.7; 491).
//
// Every mbarrier wait is bounded in time; on a time-out the CTA records a code in the status word, lets its products land, frees its
// tensor memory and returns without writing.
#include "fp4.cuh"
#include <limits.h>
#include <math.h>

namespace {

constexpr int BM = 128;                 // rows of a row tile
constexpr int QT = 2;                   // row tiles of a CTA
constexpr int BN = 128;                 // keys of a tile
constexpr int NTHREADS = 512;
constexpr int W_UNPACK = 8, W_SCORES = 12;
// Registers a thread after the trade: softmax / unpack / the rest; the sum stays within what the launch allots (128 a thread).
constexpr int REGS_SOFTMAX = 192, REGS_UNPACK = 88, REGS_REST = 40;
static_assert(QT * REGS_SOFTMAX + REGS_UNPACK + REGS_REST <= 4 * 128, "registers are traded, not made");
constexpr float LOG2E = 1.4426950408889634f;
constexpr float LAG = 6.f, BIAS = 8.f;  // how far (in powers of two) the maximum in use may lag; what the weights are raised by
constexpr int MOST_PIECES = 32;
constexpr unsigned long long WAIT_NS = 2000ull * 1000ull * 1000ull;
enum : int { ERR_UNPACK_WAIT = 321, ERR_ISSUER_WAIT = 322, ERR_SOFTMAX_WAIT = 323, ERR_PLACE = 324 };
constexpr unsigned TMEM_COLS = 512;

struct Params {
    const __nv_bfloat16* q;
    __nv_bfloat16* out;
    const unsigned char* k_pages;
    const unsigned char* v_pages;
    const int* block_table;
    const int* q_start;
    const int* kv_len;
    float* part_o;              // [row of q * n_heads + head, pieces, head_dim]
    float* part_ml;             // the same with 2: maximum (base 2) and sum of the weights
    int* status;
    long long n_pages;
    int table_stride, table_cols;
    int n_heads, n_kv_heads, group, page_records;
    int n_seqs, pieces, window;
    int most_blocks;            // of a request
    int page_shift;             // page_records is 1 << page_shift, or page_shift is negative
    unsigned per_group;         // 2^32 / group and one more (0 for a group of one head): row / group without a division
    float scale_log2;
};
// (exact for row * group < 2^32, which the host sees to)
__device__ __forceinline__ int token_of(const Params& p, int row) { return p.per_group ? (int)__umulhi((unsigned)row, p.per_group) : row; }

__device__ __forceinline__ unsigned smem_u32(const void* p) { return (unsigned)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void mbar_init(unsigned long long* bar, unsigned count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(bar)), "r"(count));
}
__device__ __forceinline__ void mbar_arrive(unsigned long long* bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ bool mbar_try_wait(unsigned long long* bar, unsigned parity) {
    unsigned ok;
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                 : "=r"(ok) : "r"(smem_u32(bar)), "r"(parity) : "memory");
    return ok != 0;
}
// false once WAIT_NS have passed, or as soon as another role has given up
__device__ __forceinline__ bool mbar_wait(unsigned long long* bar, unsigned parity, volatile int* failed) {
    if (mbar_try_wait(bar, parity)) return true;
    unsigned long long t0;
    asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t0));
    for (unsigned i = 1;; ++i) {
        if (mbar_try_wait(bar, parity)) return true;
        if ((i & 255u) == 0u) {
            unsigned long long t1;
            asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t1));
            if (*failed || t1 - t0 > WAIT_NS) return false;
        }
    }
}

// shared-memory matrix descriptors, 128-byte swizzle, rows of 128 bytes, 8-row groups 1024 bytes apart.
// K-major (Q, K, P): the row is the M or N index, K runs along the 128-byte row.
__device__ __forceinline__ unsigned long long desc_k_major(unsigned addr) {
    unsigned long long d = 0;
    d |= (unsigned long long)((addr & 0x3FFFFu) >> 4);
    d |= (unsigned long long)(1024u >> 4) << 32;                 // between 8-row groups
    d |= (unsigned long long)1u << 46;
    d |= (unsigned long long)2u << 61;
    return d;
}
// MN-major (V as stored): the 128-byte row is a key (the K index) holding 64 consecutive columns
// (the N index); 8 keys make a 1024-byte group, the next 64 columns lie block_bytes further on.
__device__ __forceinline__ unsigned long long desc_mn_major(unsigned addr, unsigned block_bytes) {
    unsigned long long d = 0;
    d |= (unsigned long long)((addr & 0x3FFFFu) >> 4);
    d |= (unsigned long long)((block_bytes >> 4) & 0x3FFFu) << 16;   // between 64-column blocks
    d |= (unsigned long long)(1024u >> 4) << 32;                     // between 8-key groups
    d |= (unsigned long long)1u << 46;
    d |= (unsigned long long)2u << 61;
    return d;
}
// instruction descriptor: float16 operands, float32 accumulator, M = 128, N = n
__host__ __device__ constexpr unsigned idesc(int n, unsigned b_mn_major) {
    return (1u << 4) | (b_mn_major << 16) | ((unsigned)(n >> 3) << 17) | ((unsigned)(BM >> 4) << 24);
}
// The three tensor-core instructions below are for a whole warp in step: one elected lane issues.  So
// the descriptors stay warp-uniform values (uniform registers); a lone lane inside a divergent branch
// cannot have those, and its instructions issued a fifth slower.
// D[tmem] (+)= A[shared] . B[shared]
__device__ __forceinline__ void umma_ss_elect(unsigned tmem_d, unsigned long long a_desc, unsigned long long b_desc,
                                              unsigned id, unsigned accumulate) {
    asm volatile("{\n\t.reg .pred p, e;\n\telect.sync _|e, 0xffffffff;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                 "@e tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
                 ::"r"(tmem_d), "l"(a_desc), "l"(b_desc), "r"(id), "r"(accumulate) : "memory");
}
// D[tmem] (+)= A[tmem] . B[shared]: the left operand lies in tensor memory, row = lane, two 16-bit
// elements of K to a column
__device__ __forceinline__ void umma_ts_elect(unsigned tmem_d, unsigned tmem_a, unsigned long long b_desc,
                                              unsigned id, unsigned accumulate) {
    asm volatile("{\n\t.reg .pred p, e;\n\telect.sync _|e, 0xffffffff;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                 "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
                 ::"r"(tmem_d), "r"(tmem_a), "l"(b_desc), "r"(id), "r"(accumulate) : "memory");
}
// the barrier gets an arrival when everything this lane has issued so far is done
__device__ __forceinline__ void umma_commit_elect(unsigned long long* bar) {
    asm volatile("{\n\t.reg .pred e;\n\telect.sync _|e, 0xffffffff;\n\t"
                 "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void tmem_ld16(unsigned taddr, unsigned (&r)[16]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
                   "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
                 : "r"(taddr));
}
__device__ __forceinline__ void tmem_st16(unsigned taddr, const unsigned (&r)[16]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
                 ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
                   "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
                 : "memory");
}
// N words (a multiple of 16) of this thread's lane, in pieces of 16 columns
template <int N> __device__ __forceinline__ void tmem_ld(unsigned taddr, unsigned (&r)[N]) {
    static_assert(N % 16 == 0, "whole pieces of 16 columns");
#pragma unroll
    for (int c = 0; c < N / 16; ++c) tmem_ld16(taddr + c * 16, *reinterpret_cast<unsigned(*)[16]>(&r[c * 16]));
}
template <int N> __device__ __forceinline__ void tmem_st(unsigned taddr, const unsigned (&r)[N]) {
    static_assert(N % 16 == 0, "whole pieces of 16 columns");
#pragma unroll
    for (int c = 0; c < N / 16; ++c) tmem_st16(taddr + c * 16, *reinterpret_cast<const unsigned(*)[16]>(&r[c * 16]));
}
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ float ex2(float x) {     // 2^x, one instruction; 2^-inf = 0
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// ones in the lowest n places (none below 0, all from 32 on)
__device__ __forceinline__ unsigned first_bits(int n) {
    unsigned m;
    asm("shr.u32 %0, 0xffffffff, %1;" : "=r"(m) : "r"(32 - min(max(n, 0), 32)));       // (a shift by 32 leaves nothing)
    return m;
}
__device__ __forceinline__ unsigned pack_bf16(float lo, float hi) {
    __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<unsigned*>(&v);
}
// 16 bytes from global to shared memory, `bytes` of them from there and zeros for the rest
__device__ __forceinline__ void copy16(void* to, const void* from, int bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(to)), "l"(from), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_all;" ::: "memory"); }
// 32 bytes, a whole sector (the address is a multiple of 32)
__device__ __forceinline__ void store32(void* to, const unsigned (&w)[8]) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(to), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]),
                 "r"(w[6]), "r"(w[7]) : "memory");
}
__device__ __forceinline__ float max3_abs(float a, float b, float c) {      // the largest magnitude; not a number if one is none
    float d;
    asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
__device__ __forceinline__ unsigned pack_half(float lo, float hi) {
    __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<unsigned*>(&v);
}

template <int KSTAGES, int VSTAGES>
struct Tail {                   // what lies behind the tiles in shared memory
    unsigned long long q_full, k_full[KSTAGES], k_empty[KSTAGES], v_full[VSTAGES], v_empty[VSTAGES];
    unsigned long long s_full[QT], s_free, p_half[QT], p_full[QT], pv_done[QT], noted, settled[2];
    unsigned tmem_base_slot;
    int failed_flag;
    // Groups of values that are not numbers, a bit each, of the keys that some rows of the CTA see and others do not: those behind the first row's
    // place, and those ahead of the last row's window.  Its rows lie within 256 places, so there are no more of either.
    int any_nan;
    unsigned char nan_late[QT * BM], nan_early[QT * BM];
};

// What a row tile has to do with the CTA's key tiles (counted from the piece's first): it works on tiles first .. last - 1.
struct TileRange {
    int rows, first, last, low, high;       // low, high: places of its first and last token in the request
};

template <int N> __device__ __forceinline__ void regs_up() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N> __device__ __forceinline__ void regs_down() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }

// A key's (or value's) numbers and scales: HD / 32 pieces of 16 bytes, HD / 16 bytes of scales.  (Plain loads: the kernel before this one may write
// the pages while a CTA is already resident, so they are not memory that nobody writes as long as this kernel runs.)
template <int HD>
struct Packed {
    uint4 codes[HD / 32];
    uint2 scales;
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < HD / 32; ++i) codes[i] = make_uint4(0u, 0u, 0u, 0u);
        scales = make_uint2(0u, 0u);
    }
    __device__ __forceinline__ void load(const unsigned char* record, int row) {
#pragma unroll
        for (int i = 0; i < HD / 32; ++i) codes[i] = *reinterpret_cast<const uint4*>(record + row * (HD / 2) + i * 16);
        const unsigned char* s = record + FP4_RECORD * (HD / 2) + row * (HD / FP4_GROUP);
        if (HD == 128) scales = *reinterpret_cast<const uint2*>(s);
        else scales.x = *reinterpret_cast<const unsigned*>(s);
    }
    // The groups that are not numbers, a bit each.
    __device__ __forceinline__ unsigned nan_groups() const {
        unsigned none = 0;
#pragma unroll
        for (int c = 0; c < HD / FP4_GROUP; ++c)
            if ((((c < 4 ? scales.x : scales.y) >> (8 * (c & 3))) & 255u) == (unsigned)FP4_NAN_SCALE) none |= 1u << c;
        return none;
    }
    // Zeros for some groups of what `unpack` has written.
    static __device__ __forceinline__ void clear_groups(unsigned char* tile, int key, unsigned groups) {
#pragma unroll 1
        for (int c = 0; c < HD / 8; ++c)
            if ((groups >> (c / 2)) & 1u)
                *reinterpret_cast<uint4*>(tile + key * 128 + (c >> 3) * (BN * 128) + (((c & 7) ^ (key & 7)) << 4)) = make_uint4(0u, 0u, 0u, 0u);
    }
    // float16 rows of 128 bytes (64 coordinates), 16-byte chunks exchanged as the 128-byte swizzle has them
    __device__ __forceinline__ void unpack(unsigned char* tile, int key) const {
        unsigned char* at = tile + key * 128;
#pragma unroll
        for (int c = 0; c < HD / 8; ++c) {
            const uint4 q = codes[c / 4];
            const unsigned w = (c & 3) == 0 ? q.x : (c & 3) == 1 ? q.y : (c & 3) == 2 ? q.z : q.w;
            const unsigned sw = c / 2 < 4 ? scales.x : scales.y;
            const __half2 s = fp4_scale2((sw >> (8 * ((c / 2) & 3))) & 255u);
            __half2 r[4];
            fp4_unpack(w, r);
            uint4 v;
            __half2 x = __hmul2(r[0], s); v.x = *reinterpret_cast<unsigned*>(&x);
            x = __hmul2(r[1], s); v.y = *reinterpret_cast<unsigned*>(&x);
            x = __hmul2(r[2], s); v.z = *reinterpret_cast<unsigned*>(&x);
            x = __hmul2(r[3], s); v.w = *reinterpret_cast<unsigned*>(&x);
            *reinterpret_cast<uint4*>(at + (c >> 3) * (BN * 128) + (((c & 7) ^ (key & 7)) << 4)) = v;
        }
    }
};

template <int HD, int KSTAGES, int VSTAGES>
__global__ void __launch_bounds__(NTHREADS, 1) attention_fp4_prefill_kernel(const Params p) {
    constexpr int HALVES = HD / 64;
    constexpr unsigned HALF_BYTES = BN * 128;
    constexpr unsigned KV_BYTES = HALVES * HALF_BYTES;
    // Tensor memory: a score buffer, which the row tiles use in turn.  (With head_dim 64 there is room for two; but then both row tiles wait for the
    // exponential unit together and leave it idle together: 3,290 cycles for 128 keys of both, so 3,080.)
    constexpr unsigned COL_S = 0, COL_P = BN, COL_O = COL_P + QT * (BN / 2);
    static_assert(COL_O + QT * HD <= TMEM_COLS, "scores, weights and accumulators must fit the tensor memory of a CTA");
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    unsigned char* Qs = smem_raw;
    unsigned char* Ks = Qs + QT * KV_BYTES;
    unsigned char* Vs = Ks + KSTAGES * KV_BYTES;
    Tail<KSTAGES, VSTAGES>& tail = *reinterpret_cast<Tail<KSTAGES, VSTAGES>*>(Vs + VSTAGES * KV_BYTES);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    if (tid == 0) {
        tail.failed_flag = 0;
        tail.any_nan = 0;
        mbar_init(&tail.q_full, 4 * QT);
        mbar_init(&tail.s_free, 4);
        mbar_init(&tail.noted, 4);
        for (int s = 0; s < KSTAGES; ++s) {
            mbar_init(&tail.k_full[s], 4);
            mbar_init(&tail.k_empty[s], QT);
        }
        for (int s = 0; s < VSTAGES; ++s) {
            mbar_init(&tail.v_full[s], 4);
            mbar_init(&tail.v_empty[s], QT);
        }
        for (int t = 0; t < QT; ++t) {
            mbar_init(&tail.s_full[t], 1);
            mbar_init(&tail.p_half[t], 4);
            mbar_init(&tail.p_full[t], 4);
            mbar_init(&tail.pv_done[t], 1);
            mbar_init(&tail.settled[t], 1);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        if ((smem_u32(smem_raw) & 1023u) != 0u) {       // (the swizzle goes by address)
            tail.failed_flag = 1;
            atomicExch(p.status, ERR_PLACE);
        }
    }
    if (tid < QT * BM) tail.nan_late[tid] = tail.nan_early[tid] = 0;
    if (warp == W_SCORES) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tail.tmem_base_slot)), "r"(TMEM_COLS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const unsigned tmem = tail.tmem_base_slot;
    int* failed = &tail.failed_flag;
    grid_launch_dependents();
    grid_dependency_wait();         // (lengths, tables, queries and the cache itself may come from the kernels before this one)

    const int per_block = p.n_kv_heads * p.pieces, index = blockIdx.x / per_block, rest = blockIdx.x - index * per_block;
    const int kvh = rest / p.pieces, piece = rest - kvh * p.pieces;
    // The blocks of all requests are numbered through; the request's that this one is (every warp for itself, 32 requests at a time)
    int b = 0, number = -1;
    for (int b0 = 0, before = 0; b0 < p.n_seqs && number < 0; b0 += 32) {
        const int mine = b0 + lane;
        const int count = mine < p.n_seqs ? min(((p.q_start[mine + 1] - p.q_start[mine]) * p.group + QT * BM - 1) / (QT * BM), p.most_blocks) : 0;
        int upto = count;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += v;
        }
        const unsigned here = __ballot_sync(0xffffffffu, before + upto > index);
        if (here) {
            const int src = __ffs(here) - 1;
            b = b0 + src;
            number = before + __shfl_sync(0xffffffffu, upto, src) - 1 - index;       // (the blocks that see most keys begin first)
        }
        before += __shfl_sync(0xffffffffu, upto, 31);
    }
    const int first_token = p.q_start[b];
    const int ql = p.q_start[b + 1] - first_token;
    const int base = p.kv_len[b] - ql;
    const int row0 = max(number, 0) * (QT * BM);
    const int all_rows = ql * p.group;
    const bool active = number >= 0 && *(volatile int*)failed == 0;
    const int last_row = min(row0 + QT * BM, all_rows) - 1;
    // keys lo .. hi - 1 of the block, and of this piece of them (whole tiles)
    int lo = p.window > 0 ? max(0, base + token_of(p, row0) - p.window + 1) : 0;
    int hi = min(base + (active ? token_of(p, last_row) : 0) + 1, p.table_cols * p.page_records * FP4_RECORD);
    int k_start = lo & ~(BN - 1);
    if (p.pieces > 1) {
        const int tiles = hi > k_start ? (hi - k_start + BN - 1) / BN : 0, each = (tiles + p.pieces - 1) / p.pieces;
        k_start += piece * each * BN;
        hi = min(hi, k_start + each * BN);
        lo = max(lo, k_start);
    }
    TileRange range[QT];
    int n_tiles = 0;
#pragma unroll
    for (int t = 0; t < QT; ++t) {
        const int r0 = row0 + t * BM;
        const int rows = active ? max(0, min(BM, all_rows - r0)) : 0;
        range[t].rows = rows;
        range[t].low = base + token_of(p, r0);
        range[t].high = base + (rows > 0 ? token_of(p, r0 + rows - 1) : 0);
        const int from = p.window > 0 ? max(lo, range[t].low - p.window + 1) : lo, to = min(hi, range[t].high + 1);
        const bool any = rows > 0 && to > from;
        range[t].first = any ? (from - k_start) / BN : 0;
        range[t].last = any ? (to - k_start + BN - 1) / BN : 0;
        n_tiles = max(n_tiles, range[t].last);
    }
    // Keys behind `late` are not seen by the CTA's first row, those ahead of `early` not by its last.  A value there that is not a number would reach rows that
    // do not see it (its weight is 0, and 0 times NaN is NaN): whoever unpacks it makes it zero and notes it, and the rows that see it get their NaN at the end.
    const int late = base + token_of(p, row0), early = p.window > 0 ? base + token_of(p, active ? last_row : row0) - p.window + 1 : INT_MIN;

    if (warp >= W_SCORES) {
        regs_down<REGS_REST>();
        if (warp < W_SCORES + 2 && n_tiles > 0) {
            // ---- issuers: one for the scores, one for the products into the accumulators; the whole warp runs
            // in step and one elected lane issues.  Both go through the key tiles in order, row tile 0 before 1.
            bool ok = true;
            if (warp == W_SCORES) {
                // S_j = Q K_j^T, as soon as the scores that lie in the buffer have been read
                constexpr unsigned id_s = idesc(BN, 0u);
                ok = __all_sync(0xffffffffu, mbar_wait(&tail.q_full, 0, failed));
                int used = 0;
                for (int j = 0; j < n_tiles && ok; ++j) {
                    const int s = j % KSTAGES;
                    ok = __all_sync(0xffffffffu, mbar_wait(&tail.k_full[s], (j / KSTAGES) & 1, failed));
                    const unsigned long long kd0 = desc_k_major(smem_u32(Ks + s * KV_BYTES));
#pragma unroll
                    for (int t = 0; t < QT; ++t) {
                        if (!ok) break;
                        if (j >= range[t].first && j < range[t].last) {
                            if (used > 0) ok = __all_sync(0xffffffffu, mbar_wait(&tail.s_free, (used - 1) & 1, failed));
                            if (!ok) break;
                            tc_fence_after();
                            const unsigned long long qd0 = desc_k_major(smem_u32(Qs + t * KV_BYTES));
#pragma unroll
                            for (int kd = 0; kd < HD / 16; ++kd) {
                                const unsigned off = ((kd / 4) * HALF_BYTES + (kd % 4) * 32) >> 4;
                                umma_ss_elect(tmem + COL_S, qd0 + off, kd0 + off, id_s, kd > 0 ? 1u : 0u);
                            }
                            umma_commit_elect(&tail.s_full[t]);
                            umma_commit_elect(&tail.k_empty[s]);
                            ++used;
                        } else if (lane == 0) {
                            mbar_arrive(&tail.k_empty[s]);          // not this tile's keys: nothing to wait for
                        }
                    }
                }
            } else {
                // O += P_j V_j, with the weights read from tensor memory: the product starts on the first half of
                // the keys while the second half's weights are still being taken.
                constexpr unsigned id_o = idesc(HD, 1u);
                for (int j = 0; j < n_tiles && ok; ++j) {
                    const int s = j % VSTAGES;
                    ok = __all_sync(0xffffffffu, mbar_wait(&tail.v_full[s], (j / VSTAGES) & 1, failed));
                    const unsigned long long vd0 = desc_mn_major(smem_u32(Vs + s * KV_BYTES), HALF_BYTES);
#pragma unroll
                    for (int t = 0; t < QT; ++t) {
                        if (!ok) break;
                        if (j >= range[t].first && j < range[t].last) {
                            const unsigned par = (j - range[t].first) & 1;
                            const unsigned d_p = tmem + COL_P + t * (BN / 2), d_o = tmem + COL_O + t * HD;
                            ok = __all_sync(0xffffffffu, mbar_wait(&tail.p_half[t], par, failed));
                            if (!ok) break;
                            tc_fence_after();
                            const unsigned acc = j > range[t].first ? 1u : 0u;
#pragma unroll
                            for (int kk = 0; kk < BN / 32; ++kk)
                                umma_ts_elect(d_o, d_p + kk * 8, vd0 + kk * (2048 >> 4), id_o, kk > 0 ? 1u : acc);
                            ok = __all_sync(0xffffffffu, mbar_wait(&tail.p_full[t], par, failed));
                            if (!ok) break;
                            tc_fence_after();
#pragma unroll
                            for (int kk = BN / 32; kk < BN / 16; ++kk)
                                umma_ts_elect(d_o, d_p + kk * 8, vd0 + kk * (2048 >> 4), id_o, 1u);
                            umma_commit_elect(&tail.pv_done[t]);
                            umma_commit_elect(&tail.v_empty[s]);
                        } else if (lane == 0) {
                            mbar_arrive(&tail.v_empty[s]);
                        }
                    }
                }
            }
            if (!ok && lane == 0 && atomicExch(failed, 1) == 0) atomicExch(p.status, ERR_ISSUER_WAIT);
            // (whoever has given up: no product may still be under way when tensor and shared memory become another CTA's)
            umma_commit_elect(&tail.settled[warp - W_SCORES]);
            int never = 0;
            mbar_wait(&tail.settled[warp - W_SCORES], 0, &never);
        }
    } else if (warp >= W_UNPACK) {
        regs_down<REGS_UNPACK>();
        // ---- unpack: a thread to a key of the tile
        const int key = tid - W_UNPACK * 32;
        const int* table = p.block_table + (size_t)b * p.table_stride;
        constexpr int RECORD = fp4_record_bytes(HD);
        // where the key of a tile lies (below 0: it is none of the keys in use, whatever lies there is not read)
        auto place = [&](int j) {
            const int kpos = k_start + j * BN + key;
            if (j >= n_tiles || kpos < lo || kpos >= hi) return -1ll;
            const int rec = kpos / FP4_RECORD, block = p.page_shift >= 0 ? rec >> p.page_shift : rec / p.page_records;
            long long page = table[block];
            if (!tl_check_page(page) || page < 0 || page >= p.n_pages) page = 0;       // (a bad page is not followed; debug builds report it)
            return ((page * p.n_kv_heads + kvh) * p.page_records + rec - block * p.page_records) * RECORD;
        };
        const int row = key & (FP4_RECORD - 1);            // (k_start is a multiple of a record)
        Packed<HD> held, coming;
        long long at = place(0), next = -1;
        coming.clear();
        if (at >= 0) coming.load(p.k_pages + at, row);
        bool ok = true;
        const int late_tile = max(late + 1 - k_start, 0) / BN, early_end = early > k_start ? (early - k_start + BN - 1) / BN : 0;
        // Keys and values go through the same instructions, and what runs rarely stands apart from the loops: together they just about fit the instruction
        // cache.  (With a loop that has a body for each, what hides values cost 2,048 tokens behind 14,001 472 -> 505 us and a prompt of 2,048
        // 45.6 -> 49, with none of it ever run; this way 480 and 47.)
#pragma unroll 1
        for (int i = 0; i < 2 * n_tiles; ++i) {
            const int j = i >> 1;
            const bool values = (i & 1) != 0;
            if (values) at = next;
            else next = place(j + 1);
            const int stages = values ? VSTAGES : KSTAGES, turn = values ? j / VSTAGES : j / KSTAGES, s = j - turn * stages;
            unsigned char* tile = (values ? Vs : Ks) + s * KV_BYTES;
            if (turn > 0 && !__all_sync(0xffffffffu, mbar_wait((values ? tail.v_empty : tail.k_empty) + s, (turn - 1) & 1, failed))) {
                ok = false;
                break;
            }
            held = coming;
            coming.clear();
            if (at >= 0) coming.load((values ? p.k_pages : p.v_pages) + at, row);
            held.unpack(tile, key);
            if (__builtin_expect(values && (j >= late_tile || j < early_end), 0)) {
                const int kpos = k_start + j * BN + key;
                const unsigned none = held.nan_groups();
                if (__builtin_expect(none != 0u && (kpos > late || kpos < early), 0)) {
                    held.clear_groups(tile, key, none);
                    if (kpos > late) tail.nan_late[kpos - late - 1] = (unsigned char)none;
                    else tail.nan_early[early - 1 - kpos] = (unsigned char)none;
                    tail.any_nan = 1;
                }
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");     // (the tensor cores read what was stored)
            __syncwarp();
            if (lane == 0) mbar_arrive((values ? tail.v_full : tail.k_full) + s);
        }
        if (lane == 0) mbar_arrive(&tail.noted);
        if (!ok && lane == 0 && atomicExch(failed, 1) == 0) atomicExch(p.status, ERR_UNPACK_WAIT);
    } else {
        regs_up<REGS_SOFTMAX>();
        // ---- softmax of row tile t: a thread to a row
        const int t = warp >> 2;
        const int sw = warp & 3;
        const int r = sw * 32 + lane;
        const unsigned lane_addr = tmem + ((unsigned)(sw * 32) << 16);
        const int rows = t ? range[1].rows : range[0].rows;
        const int first = t ? range[1].first : range[0].first, last = t ? range[1].last : range[0].last;
        const int low = t ? range[1].low : range[0].low, high = t ? range[1].high : range[0].high;
        const int tile_row0 = row0 + t * BM;
        unsigned char* stage = Qs + t * KV_BYTES;
        constexpr int CH = HD / 8;                 // lanes that share a row in global memory
        auto row_of = [&](int rr) {                // the row of q (and out) of a row of the tile
            const int token = token_of(p, tile_row0 + rr);
            return (size_t)(first_token + token) * p.n_heads + kvh * p.group + tile_row0 + rr - token * p.group;
        };
        // The warp's 32 rows of q come into shared memory, 16 bytes a lane, where the operand layout has them (zeros for rows that are
        // none), and there every thread brings its own row to float16.  (Loops, and not unrolled: this runs once, and straight code
        // would be fetched instruction by instruction; through registers and all unrolled a prompt
        // of 2,048 took 51 us, so 46.)
        float back = 0.f;
        if (n_tiles > 0) {
#pragma unroll 2
            for (int i = 0; i < CH; ++i) {
                const int rr = sw * 32 + i * (32 / CH) + lane / CH, chunk = lane % CH;
                copy16(stage + (chunk >> 3) * HALF_BYTES + rr * 128 + (((chunk & 7) ^ (rr & 7)) << 4), rr < rows ? p.q + row_of(rr) * HD + chunk * 8 : p.q,
                       rr < rows ? 16 : 0);
            }
            copies_wait();
            __syncwarp();
            auto at = [&](int c) { return reinterpret_cast<uint4*>(stage + (c >> 3) * HALF_BYTES + r * 128 + (((c & 7) ^ (r & 7)) << 4)); };
            // (the upper number of a word is read with the lower one behind it: that changes no exponent)
            float top = 0.f;
#pragma unroll 4
            for (int c = 0; c < CH; ++c) {
                const uint4 x = *at(c);
                top = max3_abs(top, __uint_as_float(x.x), __uint_as_float(x.x << 16));
                top = max3_abs(top, __uint_as_float(x.y), __uint_as_float(x.y << 16));
                top = max3_abs(top, __uint_as_float(x.z), __uint_as_float(x.z << 16));
                top = max3_abs(top, __uint_as_float(x.w), __uint_as_float(x.w << 16));
            }
            // the row's largest number goes to 2^14 .. 2^15 (exponents as float32 has them, 127 more than they mean)
            const int up = min(268 - (int)((__float_as_uint(top) & 0x7fffffffu) >> 23), 253);
            // (the scale's sign goes with the queries: larger sums are larger scores)
            const float factor = __uint_as_float((unsigned)up << 23 | (__float_as_uint(p.scale_log2) & 0x80000000u));
            back = __uint_as_float((unsigned)(254 - up) << 23);
#pragma unroll 2
            for (int c = 0; c < CH; ++c) {
                const uint4 x = *at(c);
                auto half2 = [&](unsigned w) { return pack_half(__uint_as_float(w << 16) * factor, __uint_as_float(w & 0xffff0000u) * factor); };
                *at(c) = make_uint4(half2(x.x), half2(x.y), half2(x.z), half2(x.w));
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(&tail.q_full);
        }
        const unsigned col_s = COL_S, col_p = COL_P + t * (BN / 2), col_o = COL_O + t * HD;
        // (above zero, for -inf times it: where 2^-126 stands for less, scores are below 2^-80 either way)
        const float fit = fmaxf(back * fabsf(p.scale_log2), 1.17549435e-38f);
        float m_used = -INFINITY, l_sum = 0.f;
        const int qpos = base + token_of(p, tile_row0 + (r < rows ? r : max(rows - 1, 0)));
        const float2 sc2 = make_float2(fit, fit);
        bool ok = true;
        for (int j = first; j < last; ++j) {
            const int k0 = k_start + j * BN;
            const int it = j - first, par = it & 1;
            ok = __all_sync(0xffffffffu, mbar_wait(&tail.s_full[t], par, failed));
            if (!ok) break;
            tc_fence_after();
            unsigned raw[BN];
            tmem_ld<BN>(lane_addr + col_s, raw);
            tmem_wait_ld();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&tail.s_free);      // the buffer may take the next scores
            const bool clear = k0 >= lo && k0 + BN <= hi && k0 + BN - 1 <= low && (p.window <= 0 || k0 > high - p.window);
            if (__builtin_expect(!clear, 0)) {
                const int from = max(lo, p.window > 0 ? qpos - p.window + 1 : 0) - k0, to = min(hi, qpos + 1) - k0;
#pragma unroll
                for (int w = 0; w < BN / 32; ++w) {
                    const unsigned seen = first_bits(to - 32 * w) & ~first_bits(from - 32 * w);
#pragma unroll
                    for (int i = 0; i < 32; ++i)
                        if (((seen >> i) & 1u) == 0u) raw[32 * w + i] = 0xff800000u;      // -inf
                }
            }
            float mx[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) mx[i] = fmaxf(__uint_as_float(raw[i]), __uint_as_float(raw[i + 4]));
#pragma unroll
            for (int i = 8; i < BN; i += 8)
#pragma unroll
                for (int k = 0; k < 4; ++k) mx[k] = max3(mx[k], __uint_as_float(raw[i + k]), __uint_as_float(raw[i + k + 4]));
            const float m_new = fmaxf(m_used, fmaxf(max3(mx[0], mx[1], mx[2]), mx[3]) * fit);
            const bool grow = m_new > m_used + LAG;      // also true for the first keys a row sees
            // (the weights of the key tile before have been read, and the accumulator may be touched, when its product is over)
            if (it > 0) {
                ok = __all_sync(0xffffffffu, mbar_wait(&tail.pv_done[t], (it - 1) & 1, failed));
                if (!ok) break;
                tc_fence_after();
            }
            if (__any_sync(0xffffffffu, grow)) {
                const float shrink = grow ? ex2(m_used - m_new) : 1.f;
                if (grow) m_used = m_new;
                l_sum *= shrink;
                if (it > 0) {
#pragma unroll 1
                    for (int c = 0; c < HD / 16; ++c) {
                        unsigned o[16];
                        tmem_ld16(lane_addr + col_o + c * 16, o);
                        tmem_wait_ld();
#pragma unroll
                        for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * shrink);
                        tmem_st16(lane_addr + col_o + c * 16, o);
                    }
                    tmem_wait_st();
                }
            }
            const float m_safe = m_used == -INFINITY ? 0.f : m_used - BIAS;
            const float2 nm2 = make_float2(-m_safe, -m_safe);
            float2 la = make_float2(0.f, 0.f), lb = make_float2(0.f, 0.f);
#pragma unroll
            for (int c = 0; c < BN / 32; ++c) {
                unsigned packed[16];
#pragma unroll
                for (int i = 0; i < 32; i += 4) {
                    const int k = c * 32 + i;
                    const float2 xa = __ffma2_rn(make_float2(__uint_as_float(raw[k]), __uint_as_float(raw[k + 1])), sc2, nm2);
                    const float2 xb = __ffma2_rn(make_float2(__uint_as_float(raw[k + 2]), __uint_as_float(raw[k + 3])), sc2, nm2);
                    const float2 ea = make_float2(ex2(xa.x), ex2(xa.y)), eb = make_float2(ex2(xb.x), ex2(xb.y));
                    la = __fadd2_rn(la, ea);
                    lb = __fadd2_rn(lb, eb);
                    packed[i / 2] = pack_half(ea.x, ea.y);
                    packed[i / 2 + 1] = pack_half(eb.x, eb.y);
                }
                tmem_st<16>(lane_addr + col_p + c * 16, packed);
                if (c == BN / 64 - 1) {          // half of the keys' weights are in place
                    tmem_wait_st();
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&tail.p_half[t]);
                }
            }
            l_sum += (la.x + la.y) + (lb.x + lb.y);
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&tail.p_full[t]);
        }
        // ---- the end: the last product, divide, store
        const int n = last - first;
        if (ok && n > 0) {
            ok = __all_sync(0xffffffffu, mbar_wait(&tail.pv_done[t], (n - 1) & 1, failed));
            tc_fence_after();
        }
        // the groups in which this row sees a value that was hidden
        unsigned none = 0;
        if (ok && n > 0) {
            ok = __all_sync(0xffffffffu, mbar_wait(&tail.noted, 0, failed));
            if (ok && *(volatile int*)&tail.any_nan != 0) {
                const int from = max(lo, p.window > 0 ? qpos - p.window + 1 : 0), to = min(hi, qpos + 1);
                for (int k = max(from, late + 1); k < to; ++k) none |= tail.nan_late[k - late - 1];
                for (int k = from; k < min(min(to, early), late + 1); ++k) none |= tail.nan_early[early - 1 - k];
            }
        }
        if (ok && rows > 0) {
            if (p.pieces == 1) {
                // (no sum: zeros for a row without a key; where all scores are -inf, from a query that is not finite, there is no softmax)
                const float inv = l_sum == 0.f ? (qpos >= 0 ? NAN : 0.f) : 1.f / l_sum;
                // (a thread its own row, whole sectors at a time: the rows of a group's heads lie side by side)
                __nv_bfloat16* to = p.out + row_of(r < rows ? r : 0) * HD;
#pragma unroll 1
                for (int c = 0; c < HD / 16; ++c) {
                    unsigned v[16], w[8];
#pragma unroll
                    for (int i = 0; i < 16; ++i) v[i] = 0u;
                    if (n > 0) {
                        tmem_ld16(lane_addr + col_o + c * 16, v);
                        tmem_wait_ld();
                    }
#pragma unroll
                    for (int e = 0; e < 8; ++e) w[e] = pack_bf16(__uint_as_float(v[2 * e]) * inv, __uint_as_float(v[2 * e + 1]) * inv);
                    if ((none >> c) & 1u) {
#pragma unroll
                        for (int e = 0; e < 8; ++e) w[e] = 0x7fff7fffu;
                    }
                    if (r < rows) store32(to + c * 16, w);
                }
            } else if (r < rows || n > 0) {
                const size_t row = row_of(r < rows ? r : 0) * p.pieces + piece;
                if (r < rows) {
                    p.part_ml[2 * row] = l_sum != l_sum ? NAN : n > 0 ? m_used : -INFINITY;    // (no maximum remembers a score that is not a number)
                    p.part_ml[2 * row + 1] = l_sum == 0.f && qpos >= 0 ? -1.f : l_sum;         // (a row that sees keys, here or in other pieces, but has no sum)
                }
                if (n > 0) {
#pragma unroll 1
                    for (int c = 0; c < HD / 16; ++c) {
                        unsigned v[16];
                        tmem_ld16(lane_addr + col_o + c * 16, v);
                        tmem_wait_ld();
                        if ((none >> c) & 1u) {
#pragma unroll
                            for (int i = 0; i < 16; ++i) v[i] = 0x7fffffffu;
                        }
                        if (r < rows) {
                            store32(p.part_o + row * HD + c * 16, *reinterpret_cast<const unsigned(*)[8]>(&v[0]));
                            store32(p.part_o + row * HD + c * 16 + 8, *reinterpret_cast<const unsigned(*)[8]>(&v[8]));
                        }
                    }
                }
            }
        } else if (!ok && lane == 0 && atomicExch(failed, 1) == 0) {
            atomicExch(p.status, ERR_SOFTMAX_WAIT);
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == W_SCORES) {
        __syncwarp();
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(TMEM_COLS) : "memory");
    }
}

// out[row, d] = sum_i 2^{m_i - M} o_i[d] / sum_i 2^{m_i - M} l_i,  M = max_i m_i: a warp to a row.
template <int HD>
__global__ void __launch_bounds__(128) merge_pieces_kernel(const float* __restrict__ part_o, const float* __restrict__ part_ml,
                                                           __nv_bfloat16* __restrict__ out, const int* __restrict__ q_start, int n_seqs,
                                                           int n_heads, int pieces) {
    grid_launch_dependents();
    grid_dependency_wait();
    const int lane = threadIdx.x & 31;
    const long long first = (long long)q_start[0] * n_heads, rows = (long long)q_start[n_seqs] * n_heads;
    const long long row = first + (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
    if (row >= rows) return;
    float m = -INFINITY, l = 0.f;
    if (lane < pieces) {
        const float2 ml = *reinterpret_cast<const float2*>(part_ml + (row * pieces + lane) * 2);
        m = ml.x;
        l = ml.y;
    }
    float M = m;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const float other = __shfl_xor_sync(0xffffffffu, M, o);
        M = (M != M || other != other) ? NAN : fmaxf(M, other);
    }
    const float f = m == -INFINITY ? 0.f : exp2f(m - M);
    const float den = warp_sum(f * l);
    const float inv = M == -INFINITY ? (__any_sync(0xffffffffu, l < 0.f) ? NAN : 0.f) : 1.f / den;        // (zeros for a row without a key)
    constexpr int N = HD / 32;
    float num[N];
#pragma unroll
    for (int i = 0; i < N; ++i) num[i] = 0.f;
    for (int s = 0; s < pieces; ++s) {
        if (__shfl_sync(0xffffffffu, m, s) == -INFINITY) continue;             // (nothing was left there)
        const float w = __shfl_sync(0xffffffffu, f, s);
        const float* o = part_o + (row * pieces + s) * HD + lane * N;
#pragma unroll
        for (int i = 0; i < N; i += 2) {
            const float2 v = *reinterpret_cast<const float2*>(o + i);
            num[i] = fmaf(w, v.x, num[i]);
            num[i + 1] = fmaf(w, v.y, num[i + 1]);
        }
    }
#pragma unroll
    for (int i = 0; i < N; i += 2)
        *reinterpret_cast<__nv_bfloat162*>(out + row * HD + lane * N + i) = __floats2bfloat162_rn(num[i] * inv, num[i + 1] * inv);
}

// ---- host side ---------------------------------------------------------------------------------

template <int HD> constexpr int k_stages_for() { return HD == 128 ? 3 : 4; }
template <int HD> constexpr int v_stages_for() { return HD == 128 ? 2 : 4; }
template <int HD> constexpr size_t smem_for() {
    return (size_t)(QT + k_stages_for<HD>() + v_stages_for<HD>()) * (HD / 64) * BN * 128 + sizeof(Tail<k_stages_for<HD>(), v_stages_for<HD>()>);
}
static_assert(smem_for<128>() <= 227 * 1024 && smem_for<64>() <= 227 * 1024, "a CTA has 227 KB of shared memory");

bool takes(int n_heads, int n_kv_heads, int head_dim, int page_size) {
    if (head_dim != 64 && head_dim != 128) return false;
    if (n_heads <= 0 || n_kv_heads <= 0 || n_heads % n_kv_heads != 0) return false;
    return page_size >= FP4_RECORD && page_size % FP4_RECORD == 0;
}

struct Plan {
    long long of_request, blocks;       // blocks of a request, of all: at most
    int pieces;
};
Plan make_plan(long long q_rows, int n_seqs, int n_heads, int n_kv_heads, int max_q_len, int max_kv_len) {
    Plan pl;
    const long long group = n_heads / n_kv_heads, rows = max_q_len * group;
    pl.of_request = (rows + QT * BM - 1) / (QT * BM);
    pl.blocks = pl.of_request * n_seqs;
    if (q_rows * group / (QT * BM) + n_seqs < pl.blocks) pl.blocks = q_rows * group / (QT * BM) + n_seqs;
    pl.pieces = 1;
    // CTAs run in waves of 148, one an SM.  A piece takes as long as its tiles and about five more (the queries, the first and
    // the last tile's way through the roles, the results); the sums of pieces cost writing and adding up.
    const long long ctas = pl.blocks * n_kv_heads;
    const int tiles = (max_kv_len + BN - 1) / BN;
    double best = 1e30;
    for (int s = 1; s <= MOST_PIECES && s <= tiles; ++s) {
        const double waves = (double)((ctas * s + 147) / 148);
        const double cost = waves * ((tiles + s - 1) / s + 5) + (s > 1 ? 4 + 0.02 * s * (double)(q_rows * group < rows * n_seqs ? q_rows * group : rows * n_seqs) * n_kv_heads / 148.0 / 16.0 : 0.0);
        if (cost < best - 1e-9) {
            best = cost;
            pl.pieces = s;
        }
    }
    return pl;
}

template <int HD> int launch(const Params& p, dim3 grid, cudaStream_t s) {
    constexpr size_t smem = smem_for<HD>();
    auto kern = attention_fp4_prefill_kernel<HD, k_stages_for<HD>(), v_stages_for<HD>()>;
    static bool raised = false;
    if (!raised) {
        cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (e != cudaSuccess) return (int)e;
        raised = true;
    }
    return (int)tl_launch(kern, grid, dim3(NTHREADS), smem, s, p);
}

}  // namespace

// workspace_floats: scratch of a call (0: none); q_rows: rows of q, all of them.
extern "C" int tl_attention_fp4_prefill_plan(long long q_rows, int n_seqs, int n_heads, int n_kv_heads, int head_dim, int max_q_len, int max_kv_len,
                                             int allow_split, int* pieces, long long* workspace_floats) {
    if (!takes(n_heads, n_kv_heads, head_dim, FP4_RECORD) || max_q_len < 1 || n_seqs < 1) return TL_BAD_SIZE;
    const Plan pl = make_plan(q_rows, n_seqs, n_heads, n_kv_heads, max_q_len, max_kv_len);
    *pieces = allow_split > 1 ? (allow_split < MOST_PIECES ? allow_split : MOST_PIECES) : allow_split ? pl.pieces : 1;
    *workspace_floats = *pieces > 1 ? q_rows * n_heads * *pieces * (head_dim + 2) : 0;
    return TL_OK;
}

// q, out: [q_rows, n_heads, head_dim] bfloat16; pages: [n_pages, n_kv_heads, page_size / 16, 9 head_dim] bytes; block_table: [n_seqs,
// table_cols] with rows table_stride apart; q_start may count from anywhere in q; pieces as the plan says.
extern "C" int tl_attention_fp4_prefill(const void* q, const void* k_pages, const void* v_pages, void* out, const int* block_table,
                                        int table_stride, int table_cols, const int* q_start, const int* kv_len, float* workspace, int* status,
                                        long long q_rows, int n_seqs, int n_heads, int n_kv_heads, int head_dim, int page_size, long long n_pages,
                                        int max_q_len, int window, float scale, int pieces, void* stream) {
    if (n_seqs <= 0 || max_q_len <= 0) return TL_OK;
    if (!takes(n_heads, n_kv_heads, head_dim, page_size) || n_pages <= 0 || pieces < 1 || pieces > MOST_PIECES || !fp4_places_fit(table_cols, page_size, max_q_len))
        return TL_BAD_SIZE;
    // (results are stored 32 bytes at a time)
    auto aligned32 = [](const void* x) { return (reinterpret_cast<uintptr_t>(x) & 31u) == 0; };
    if (!aligned16(q) || !aligned32(out) || !aligned16(k_pages) || !aligned16(v_pages) || status == nullptr) return TL_BAD_ALIGN;
    if (pieces > 1 && (workspace == nullptr || !aligned32(workspace))) return TL_BAD_SIZE;
    const Plan pl = make_plan(q_rows, n_seqs, n_heads, n_kv_heads, max_q_len, 1);
    if ((double)pl.blocks * n_kv_heads * pieces >= 2147483647.0) return TL_BAD_SIZE;
    Params p;
    p.q = (const __nv_bfloat16*)q; p.out = (__nv_bfloat16*)out;
    p.k_pages = (const unsigned char*)k_pages; p.v_pages = (const unsigned char*)v_pages;
    p.block_table = block_table; p.q_start = q_start; p.kv_len = kv_len; p.status = status; p.n_pages = n_pages;
    p.table_stride = table_stride; p.table_cols = table_cols; p.n_heads = n_heads; p.n_kv_heads = n_kv_heads; p.group = n_heads / n_kv_heads;
    p.page_records = page_size / FP4_RECORD; p.n_seqs = n_seqs; p.most_blocks = (int)pl.of_request; p.pieces = pieces; p.window = fp4_window(window, table_cols, page_size);
    p.page_shift = -1;
    for (int i = 0; i < 31; ++i)
        if (p.page_records == 1 << i) p.page_shift = i;
    p.per_group = p.group == 1 ? 0u : (unsigned)((1ull << 32) / (unsigned)p.group) + 1u;
    if ((double)pl.of_request * QT * BM * p.group >= 4294967296.0) return TL_BAD_SIZE;
    p.scale_log2 = scale * LOG2E;
    p.part_o = workspace;
    p.part_ml = pieces > 1 ? workspace + q_rows * n_heads * pieces * head_dim : nullptr;
    cudaStream_t s = (cudaStream_t)stream;
    const dim3 grid((unsigned)(pl.blocks * n_kv_heads * pieces));
    const int rc = head_dim == 128 ? launch<128>(p, grid, s) : launch<64>(p, grid, s);
    if (rc != TL_OK || pieces == 1) return rc;
    const unsigned merge = (unsigned)((q_rows * n_heads + 3) / 4);
    if (head_dim == 128)
        return (int)tl_launch(merge_pieces_kernel<128>, dim3(merge), dim3(128), 0, s, (const float*)p.part_o, (const float*)p.part_ml, p.out, q_start,
                              n_seqs, n_heads, pieces);
    return (int)tl_launch(merge_pieces_kernel<64>, dim3(merge), dim3(128), 0, s, (const float*)p.part_o, (const float*)p.part_ml, p.out, q_start, n_seqs,
                          n_heads, pieces);
}
