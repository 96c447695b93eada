// Attention over a paged cache of 4-bit keys and values (fp4.cuh) on the mma.sync tensor cores, head_dim 64 or 128: steps whose
// requests bring one token or a few, and float32 steps of any length.
//
//     o[t, h] = sum_j w_j v_j / sum_j w_j,  w_j = exp(scale q[t, h] . k_j),  j <= pos(t), j > pos(t) - window
//
// Bound by reading the cache once (144 bytes a key and head of 128, against 512 in bfloat16), and next to that by issuing the
// instructions that unpack it: 16 keys and values of 128 numbers are 64 conversions and 64 products with scales a warp, beside
// 16 products of the tensor cores.  So:
//   - The cache comes in whole records of 16 tokens by cp.async.bulk, 128 keys a stage, into a ring that a producer warp keeps
//     full across the borders of requests; four consumer warps take two records of keys and of values each, with one turn of the softmax for both.
//   - Nothing is unpacked into shared memory.  The products are taken transposed, scores^T = K Q^T and out^T = V^T P^T, so that
//     keys and values are the left operands: a lane loads the coordinates that its fragments hold (any fixed order of the
//     contraction's index will do, so they are neighbours in a row), converts them in registers, and for V exchanges half bytes of two
//     tokens first.  A cached number times its scale is a float16 exactly (fp4.cuh).
//   - Queries are brought to float16 by a power of two for each row that puts its largest number just below 2^15: no rounding for
//     bfloat16 (but of numbers 2^-31 of the largest).  float32 queries and the probabilities of float32 steps are two float16, value and remainder (22
//     bits), and their products are added up in registers, tile by tile, rounded to nearest (the tensor cores cut).
//   - Probabilities of bfloat16 steps are one float16 each (2^-12; the result's own rounding is 2^-9).
//
// Who does what: the rows of a request (token x query heads of a key head) are cut into blocks of 8 NT; the keys that a block sees, in
// tiles of 128, are laid on one line, block after block and key head after key head, with the worth of one or two tiles in front of each
// for what it costs to begin and end one, and every CTA takes an even stretch of the line, found on the device from the
// requests' lengths.  Where a block is cut, each part leaves its sums, and the CTA that is last to finish adds them up in
// order (a counter for each block and head): the result does not depend on who that is.
// In float32 steps of many rows a block has 64 of them, 16 to a consumer warp, which then takes all records of a tile: nothing is exchanged
// between the warps, and a copied tile serves four times the rows.
// Every wait is bounded; a CTA whose wait runs out sets the status word and takes part in the counting only.
//
// Measured (32 / 8 heads, us; a record's arithmetic is 427 cycles of a scheduler, 12 consumer warps an SM):
//   bfloat16, heads of 128: 8 requests of 2,049 tokens 12.0 (19 MB; of it finding the stretch and fetching queries 2, joining warps and parts 3); 64 of 200
//   to 16,000 147 to 158 from box to box (651 MB, 4.1 to 4.4 TB/s; the copies alone 113, unpacking alone some 104); 4 of 27,001 to 32,767 36.9 (134 MB, 3.6
//   TB/s: DRAM at 42 %, unpacking alone some 22 us).  Neither copies nor unpacking bound these two by themselves: they do not hide each other.
//   One request of 333, heads of 64: 7.6, a launch and a chain of trips to memory.
//   float32, heads of 64: 12 requests of 2 to 4 tokens in a window of 1,024 15.3; prompts of 500 to 901 tokens 58.3 (16 rows a block: 73, half
//   of it beginning blocks and exchanging results).  float32 blocks of 16 rows and more with heads of 128 want more than the 168 registers that two CTAs
//   an SM leave a thread: some 600 bytes of spills (8 requests of 512 tokens behind 4,000: 2.3 ms).
#include "fp4.cuh"
#include <limits.h>
#include <math.h>

namespace {

constexpr int NCW = 4;                  // consumer warps
constexpr int EACH = 2;                 // records that a consumer warp takes of a tile: one turn of the softmax for both
constexpr int RECORDS = EACH * NCW;     // records of a tile
constexpr int BN = RECORDS * FP4_RECORD;
constexpr int NTHREADS = (NCW + 1) * 32;
constexpr int MOST_PARTS = 64;          // parts of a block, at most
// A CTA's stretch, at least.  (32 / 8 heads of 128, three and two, us: 1 request of 500 tokens 9.1 8.3, 2 of 1,000 9.5 8.8, 8 of 700 11.2 10.5, 16 of 400 11.6
// 10.6; 1 of 333 with heads of 64 7.3 7.5; a single key head, whose parts are then many, 1 of 8,000 13.1 14.3.  One is as two.)
constexpr int LEAST = 2;
constexpr int FAILED_PART = 1 << 16;    // what a CTA that gave up adds to a counter beside its 1
constexpr int SMS = 148;
constexpr float LOG2E = 1.4426950408889634f;
// The maximum that exponents are taken against may lag behind by a factor of up to 2^LAG: then no lane asks another for its
// maximum.  Weights are multiplied as 2^BIAS times what they are: as float16, down to 2^-34 of the largest.
constexpr float LAG = 4.f, BIAS = 11.f;
constexpr unsigned long long WAIT_NS = 2000ull * 1000ull * 1000ull;
enum : int { ERR_PRODUCER_WAIT = 221, ERR_CONSUMER_WAIT = 222, ERR_COUNT = 223 };

struct Params {
    const void* q;
    void* out;
    const unsigned char* k_pages;
    const unsigned char* v_pages;
    const int* block_table;
    const int* q_start;
    const int* kv_len;
    float* part;                // [CTAs, 2, part_floats]: rows x HD sums, then maximum (base 2) and sum of the weights of every row
    int* counters;              // [n_seqs, blocks, n_kv_heads], zero between launches
    int* status;
    long long n_pages;
    int table_stride, table_cols, n_seqs, n_heads, n_kv_heads, group, page_records, blocks, rows, window;
    unsigned per_group;         // 2^32 / group and one more (0 for a group of one head): row / group without a division
    int page_shift;             // page_records is 1 << page_shift, or page_shift is negative
    float scale_log2;
};

// floats of a part: whole 16 bytes also for an odd number of rows, since sums are stored four at a time
__host__ __device__ constexpr int part_floats(int rows, int head_dim) { return (rows * (head_dim + 2) + 3) / 4 * 4; }

__device__ __forceinline__ unsigned smem_u32(const void* p) { return (unsigned)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void mbar_init(unsigned long long* bar, unsigned count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(bar)), "r"(count));
}
__device__ __forceinline__ void mbar_expect_tx(unsigned long long* bar, unsigned bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_u32(bar)), "r"(bytes) : "memory");
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
__device__ __forceinline__ bool mbar_wait(unsigned long long* bar, unsigned parity, const volatile int* failed) {
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
// The wait of a whole warp: false for all lanes if it ran out for any.  The first in the CTA to give up reports.
__device__ __forceinline__ bool warp_wait(unsigned long long* bar, unsigned parity, int* failed_flag, int* status, int code, int lane) {
    if (__all_sync(0xffffffffu, mbar_wait(bar, parity, failed_flag))) return true;
    if (lane == 0 && atomicExch(failed_flag, 1) == 0) atomicExch(status, code);
    return false;
}
// (both addresses and the size are multiples of 16: records are)
__device__ __forceinline__ void bulk_load(void* dst, const void* src, unsigned bytes, unsigned long long* bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 ::"r"(smem_u32(dst)), "l"(src), "r"(bytes), "r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void mma_f16(float (&d)[4], const unsigned (&a)[4], unsigned b0, unsigned b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float ex2(float x) {     // 2^x, one instruction; 2^-inf = 0
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
__device__ __forceinline__ unsigned bits(__half2 h) { return *reinterpret_cast<unsigned*>(&h); }
__device__ __forceinline__ unsigned select_bits(unsigned mask, unsigned x, unsigned y) {      // x where mask is set, else y: one instruction
    unsigned d;
    asm("lop3.b32 %0, %1, %2, %3, 0xca;" : "=r"(d) : "r"(mask), "r"(x), "r"(y));
    return d;
}
// (shifts as products: multiply-adds have a pipe of their own, shifts share the conversions')
__device__ __forceinline__ unsigned mad(unsigned a, unsigned b, unsigned c) {
    unsigned d;
    asm("mad.lo.u32 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
    return d;
}
__device__ __forceinline__ unsigned movmatrix_trans(unsigned a) {     // 8 x 8 block of 16-bit numbers, transposed across the warp
    unsigned d;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
    return d;
}
// ones in the lowest n places (none below 0, all from 32 on)
__device__ __forceinline__ unsigned first_bits(int n) {
    unsigned m;
    asm("shr.u32 %0, 0xffffffff, %1;" : "=r"(m) : "r"(32 - min(max(n, 0), 32)));       // (a shift by 32 leaves nothing)
    return m;
}
__device__ __forceinline__ void consumers_sync() { asm volatile("bar.sync 1, %0;" ::"n"(NCW * 32) : "memory"); }

// (exact for row * group < 2^32, which the host sees to)
__device__ __forceinline__ int token_of(const Params& p, int row) { return p.per_group ? (int)__umulhi((unsigned)row, p.per_group) : row; }

// ---- the line of tiles
// What a block's beginning and end are worth, in tiles: a tile of 64 rows is four times the work of one of 16.  (8 requests of 32,000 tokens 37.0 us
// with 1 and 35.9 with 2, a 32-bit prompt of 16 rows a block 79 and 73; with 64 rows a block 56.0 with 1 and 58.5 with 2.)
__host__ __device__ constexpr int worth_of(int rows) { return rows > 16 ? 1 : 2; }
// What a block of a request's rows sees.
struct Block {
    int b, number;
    int first;          // the row of q of the request's first new token
    int base;           // that token's place in the request
    int row0, n_rows;   // rows row0 .. of the request: row = token * group + head of the group
    int lo, hi;         // visible keys lo .. hi - 1 (of any of the rows)
    int start, tiles;   // its tiles: the first begins at key `start`, on a record
};
template <int ROWS> __device__ __forceinline__ int block_at(const Params& p, int i, Block& k) {      // its worth of one key head, 0: there is no such block
    k.b = p.blocks == 1 ? i : i / p.blocks;
    k.number = i - k.b * p.blocks;
    k.first = p.q_start[k.b];
    const int ql = p.q_start[k.b + 1] - k.first;
    k.row0 = k.number * ROWS;
    // (p.rows, fewer than ROWS where one block has all: a request that brings more tokens than the step's max_q_len must not have
    // rows that the places of the warps' and parts' results were not made for.  With ROWS beside it the compiler knows a bound: one token 7.66 -> 7.54 us)
    k.n_rows = min(min(ROWS, ql * p.group - k.row0), p.rows);
    if (k.n_rows <= 0) return 0;
    k.base = p.kv_len[k.b] - ql;
    const int t0 = token_of(p, k.row0), t1 = token_of(p, k.row0 + k.n_rows - 1);
    k.lo = p.window > 0 ? max(0, k.base + t0 - p.window + 1) : 0;
    k.hi = min(k.base + t1 + 1, p.table_cols * p.page_records * FP4_RECORD);
    k.start = k.lo & ~(FP4_RECORD - 1);
    k.tiles = max((k.hi - k.start + BN - 1) / BN, 1);
    return k.tiles + worth_of(ROWS);
}
// A CTA's way along its stretch: parts of blocks, one after the other.
struct Walk {
    Block k;
    int i, kvh;
    int off;            // place on the line where (block, kvh) begins
    int begin, end, share;
    int t0, t1;         // the tiles of the part
    int parts;          // in how many parts the block is cut (for this head)
};
template <int ROWS> __device__ __forceinline__ bool walk_here(const Params& p, Walk& w) {      // the part of the place where w stands; false: beyond the stretch
    if (w.off + worth_of(ROWS) >= w.end) return false;
    w.t0 = max(0, w.begin - w.off - worth_of(ROWS));
    w.t1 = min(w.k.tiles, w.end - w.off - worth_of(ROWS));
    w.parts = w.t1 - w.t0 == w.k.tiles ? 1 : (w.off + worth_of(ROWS) + w.k.tiles - 1) / w.share - (w.off + worth_of(ROWS)) / w.share + 1;
    return true;
}
template <int ROWS> __device__ __forceinline__ bool walk_next(const Params& p, Walk& w) {
    w.off += w.k.tiles + worth_of(ROWS);
    if (++w.kvh == p.n_kv_heads) {
        w.kvh = 0;
        do {
            if (++w.i >= p.n_seqs * p.blocks) return false;
        } while (block_at<ROWS>(p, w.i, w.k) == 0);
    }
    return walk_here<ROWS>(p, w);
}
template <int ROWS> __device__ __forceinline__ bool walk_first(const Params& p, Walk& w, int lane) {
    const int n = p.n_seqs * p.blocks;
    int total = 0, longest = 0, mine = 0;
    for (int i = lane; i < n; i += 32) {
        Block k;
        mine = block_at<ROWS>(p, i, k);
        total += mine;
        longest = max(longest, mine);
    }
    total = __reduce_add_sync(0xffffffffu, total) * p.n_kv_heads;
    longest = __reduce_max_sync(0xffffffffu, longest);
    w.share = max(max((total + (int)gridDim.x - 1) / (int)gridDim.x, (longest + MOST_PARTS - 2) / (MOST_PARTS - 1)), LEAST);
    w.begin = blockIdx.x * w.share;
    w.end = w.begin + w.share;
    if (w.begin >= total) return false;
    int before = 0;                                     // worth (of all heads) of the blocks before these 32
    for (int i0 = 0; i0 < n; i0 += 32) {
        if (n > 32) {                                   // (up to 32 blocks: each lane still has its own)
            Block k;
            mine = i0 + lane < n ? block_at<ROWS>(p, i0 + lane, k) : 0;
        }
        int upto = mine * p.n_kv_heads;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += v;
        }
        const unsigned here = __ballot_sync(0xffffffffu, before + upto > w.begin);
        if (here) {
            const int src = __ffs(here) - 1;            // the first block that reaches beyond the stretch's beginning
            w.i = i0 + src;
            const int worth = block_at<ROWS>(p, w.i, w.k);
            const int at = before + __shfl_sync(0xffffffffu, upto, src) - worth * p.n_kv_heads;
            w.kvh = (w.begin - at) / worth;
            w.off = at + w.kvh * worth;
            return walk_here<ROWS>(p, w);
        }
        before += __shfl_sync(0xffffffffu, upto, 31);
    }
    return false;
}

// Two numbers as a pair of float16, and what is left of them as another.
__device__ __forceinline__ void split2(float x, float y, unsigned& hi, unsigned& lo) {
    const __half2 h = __floats2half2_rn(x, y);
    const float2 back = __half22float2(h);
    hi = bits(h);
    lo = bits(__floats2half2_rn(x - back.x, y - back.y));
}

__device__ __forceinline__ void load_row(const __nv_bfloat16* p, float (&x)[8]) {
    Vec16<__nv_bfloat16> v;
    v.load(p);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = v.get(i);
}
__device__ __forceinline__ void load_row(const float* p, float (&x)[8]) {
    Vec16<float> a, b;
    a.load(p);
    b.load(p + 4);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        x[i] = a.get(i);
        x[i + 4] = b.get(i);
    }
}
__device__ __forceinline__ void store4(__nv_bfloat16* p, float4 v) {
    const __nv_bfloat162 a = __floats2bfloat162_rn(v.x, v.y), b = __floats2bfloat162_rn(v.z, v.w);
    *reinterpret_cast<uint2*>(p) = make_uint2(*reinterpret_cast<const unsigned*>(&a), *reinterpret_cast<const unsigned*>(&b));
}
__device__ __forceinline__ void store4(float* p, float4 v) { *reinterpret_cast<float4*>(p) = v; }

// What a consumer warp keeps of a block.  Lane (g, t) = (lane / 4, lane % 4).  Of the scores^T tile it holds keys g and g + 8 for rows
// 2t and 2t + 1 of every eight, of the out^T tile coordinates HD / 8 * g + 2m and + 1 for the same rows.  Its part of a key or
// query is coordinates HD / 4 * t and the HD / 4 - 1 after them.
template <typename T, int HD, int NT, bool UNEVEN>
struct Consumer {
    static constexpr int PARTS = sizeof(T) == 4 ? 2 : 1;
    static constexpr int KSTEPS = HD / 16, WORDS = HD / 32, ROWS = 8 * NT, OPITCH = HD + 4;
    unsigned qf[PARTS][NT][KSTEPS][2];
    float fit[NT][2];                   // scale * log2(e) over the power of two that a row's queries were multiplied by
    float m[NT][2], l[NT][2], o[NT][KSTEPS][4];
    int qpos[NT][2], qmax, qmin;
    int g, t;
    unsigned spoilt;                    // rows (a bit each) that see a value of this lane's coordinates which is not a number and was hidden

    __device__ __forceinline__ void begin(const Params& p, const Block& k, int kvh, int lane) {
        g = lane >> 2;
        t = lane & 3;
        spoilt = 0;
        int top_pos = -1, low_pos = INT_MAX;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const int r = nt * 8 + g;
            const int row = k.row0 + r, token = token_of(p, row);
            float x[WORDS][8];
            unsigned top = 0;
#pragma unroll
            for (int j = 0; j < WORDS; ++j) {
#pragma unroll
                for (int i = 0; i < 8; ++i) x[j][i] = 0.f;
                if (r < k.n_rows)
                    load_row(reinterpret_cast<const T*>(p.q) + ((size_t)(k.first + token) * p.n_heads + kvh * p.group + row - token * p.group) * HD +
                                 t * (HD / 4) + j * 8, x[j]);
#pragma unroll
                for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(x[j][i]) & 0x7fffffffu);
            }
            top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
            // the row's largest number goes to 2^14 .. 2^15 (exponents as float32 has them, 127 more than they mean)
            const int up = min(268 - (int)(top >> 23), 253);
            // (the scale's sign goes with the queries, so that larger sums are larger scores; and what scores are multiplied by stays above
            // zero, for -inf times it: where 2^-126 stands for less, scores are below 2^-80 either way)
            const float factor = __uint_as_float((unsigned)up << 23 | (__float_as_uint(p.scale_log2) & 0x80000000u));
            const float back = fmaxf(__uint_as_float((unsigned)(254 - up) << 23) * fabsf(p.scale_log2), 1.17549435e-38f);
#pragma unroll
            for (int j = 0; j < WORDS; ++j)
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const float a = x[j][4 * h + 2 * e] * factor, c = x[j][4 * h + 2 * e + 1] * factor;
                        if (PARTS == 2)
                            split2(a, c, qf[0][nt][2 * j + h][e], qf[PARTS - 1][nt][2 * j + h][e]);
                        else
                            qf[0][nt][2 * j + h][e] = bits(__floats2half2_rn(a, c));
                    }
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                fit[nt][j] = __shfl_sync(0xffffffffu, back, (2 * t + j) * 4);
                const int rr = nt * 8 + 2 * t + j;
                qpos[nt][j] = rr < k.n_rows ? k.base + token_of(p, k.row0 + rr) : -1;
                top_pos = max(top_pos, qpos[nt][j]);
                if (rr < k.n_rows) low_pos = min(low_pos, qpos[nt][j]);
                m[nt][j] = -INFINITY;
                l[nt][j] = 0.f;
            }
#pragma unroll
            for (int i = 0; i < KSTEPS; ++i) o[nt][i][0] = o[nt][i][1] = o[nt][i][2] = o[nt][i][3] = 0.f;
        }
        qmax = __reduce_max_sync(0xffffffffu, top_pos);
        qmin = __reduce_min_sync(0xffffffffu, low_pos);
    }

    // numbers of a row, `WORDS` words, under their scales
    static __device__ __forceinline__ void load_words(const unsigned char* at, unsigned (&w)[WORDS]) {
        if (WORDS == 4) {
            const uint4 v = *reinterpret_cast<const uint4*>(at);
            w[0] = v.x; w[1] = v.y; w[WORDS - 2] = v.z; w[WORDS - 1] = v.w;
        } else {
            const uint2 v = *reinterpret_cast<const uint2*>(at);
            w[0] = v.x; w[1] = v.y;
        }
    }

    // A value that is not a number would reach rows that do not see it (its weight is 0, and 0 times NaN is NaN).  So those of a record, whose first key
    // is k, take part as zeros where some rows see a key and others do not, and the rows that see one are remembered.  byte: scales of this lane's
    // coordinates of four keys; the lanes that share g have the same coordinates, for other rows, and the other keys.
    __device__ __forceinline__ void hide_nan(const Params& p, unsigned (&byte)[4], int k) {
        unsigned keys = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (byte[i] == FP4_NAN_SCALE) {
                keys |= 1u << (2 * t + (i & 1) + 8 * (i >> 1));
                byte[i] = 0;
            }
        keys |= __shfl_xor_sync(0xffffffffu, keys, 1);
        keys |= __shfl_xor_sync(0xffffffffu, keys, 2);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int from = p.window > 0 ? qpos[nt][j] + 1 - p.window - k : 0;
                if (keys & first_bits(qpos[nt][j] + 1 - k) & ~first_bits(from)) spoilt |= 1u << (2 * nt + j);
            }
    }
    // When the keys are through: what was hidden of the rows that see it.
    __device__ __forceinline__ void spoil() {
        if (!__any_sync(0xffffffffu, spoilt != 0u)) return;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int j = 0; j < 2; ++j)
                if ((spoilt >> (2 * nt + j)) & 1u) {
#pragma unroll
                    for (int d = 0; d < KSTEPS; ++d) o[nt][d][j] = o[nt][d][j + 2] = NAN;
                }
    }

    // EACH records of keys and of values, APART records apart; the first begins with key k0
    template <int APART> __device__ __forceinline__ void records(const Params& p, const unsigned char* kr, const unsigned char* vr, int k0, int lo, int hi) {
        constexpr int CODES = FP4_RECORD * (HD / 2);            // where a record's scales begin
        constexpr int RECORD = fp4_record_bytes(HD), STEP = APART * FP4_RECORD, SPAN = (EACH - 1) * STEP + FP4_RECORD;
        if (k0 > qmax || k0 + SPAN <= lo || k0 >= hi) return;
        if (APART == 1 && p.window > 0 && k0 + SPAN - 1 <= qmin - p.window) return;     // (the first key of a block is the first row's)
        // ---- scores
        float sc[EACH][NT][4];
#pragma unroll
        for (int n = 0; n < EACH; ++n) {
            const unsigned char* rec = kr + n * APART * RECORD;
            float low[NT][4];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int e = 0; e < 4; ++e) sc[n][nt][e] = low[nt][e] = 0.f;
            unsigned wa[WORDS], wb[WORDS];
            load_words(rec + g * (HD / 2) + t * (HD / 8), wa);
            load_words(rec + (g + 8) * (HD / 2) + t * (HD / 8), wb);
            __half2 sa[WORDS / 2], sb[WORDS / 2];                   // a scale for two words
            if (HD == 128) {
                sa[0] = fp4_scale2(rec[CODES + g * 8 + 2 * t]); sa[WORDS / 2 - 1] = fp4_scale2(rec[CODES + g * 8 + 2 * t + 1]);
                sb[0] = fp4_scale2(rec[CODES + (g + 8) * 8 + 2 * t]); sb[WORDS / 2 - 1] = fp4_scale2(rec[CODES + (g + 8) * 8 + 2 * t + 1]);
            } else {
                sa[0] = fp4_scale2(rec[CODES + g * 4 + t]);
                sb[0] = fp4_scale2(rec[CODES + (g + 8) * 4 + t]);
            }
#pragma unroll
            for (int j = 0; j < WORDS; ++j) {
                __half2 a[4], c[4];
                fp4_unpack(wa[j], a);
                fp4_unpack(wb[j], c);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    a[i] = __hmul2(a[i], sa[j / 2]);
                    c[i] = __hmul2(c[i], sb[j / 2]);
                }
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const unsigned f[4] = {bits(a[2 * h]), bits(c[2 * h]), bits(a[2 * h + 1]), bits(c[2 * h + 1])};
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        if (PARTS == 2) {
                            float s[4] = {0.f, 0.f, 0.f, 0.f};
                            mma_f16(s, f, qf[0][nt][2 * j + h][0], qf[0][nt][2 * j + h][1]);
                            mma_f16(low[nt], f, qf[PARTS - 1][nt][2 * j + h][0], qf[PARTS - 1][nt][2 * j + h][1]);
#pragma unroll
                            for (int e = 0; e < 4; ++e) sc[n][nt][e] += s[e];
                        } else {
                            mma_f16(sc[n][nt], f, qf[0][nt][2 * j + h][0], qf[0][nt][2 * j + h][1]);
                        }
                    }
                }
            }
            if (PARTS == 2) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int e = 0; e < 4; ++e) sc[n][nt][e] += low[nt][e];
            }
        }
        // ---- masks
        const bool inside = k0 >= lo && k0 + SPAN <= hi;
        const bool clear = inside && k0 + SPAN - 1 <= qmin && (p.window <= 0 || k0 > qmax - p.window);     // (every row sees every key)
        if (!clear) {
#pragma unroll
            for (int n = 0; n < EACH; ++n)
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int qp = qpos[nt][e & 1], kpos = k0 + n * STEP + g + 8 * (e >> 1);
                        if (!(kpos >= lo && kpos < hi && kpos <= qp && (p.window <= 0 || kpos > qp - p.window))) sc[n][nt][e] = -INFINITY;
                    }
        }
        // ---- weights, moved from result layout [key g][rows 2t, 2t + 1] to operand layout [keys 2t, 2t + 1][row g]
        unsigned ph[EACH][NT][2], pl[EACH][NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            float mx[2];
            bool grown = false;
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                mx[j] = fmaxf(sc[0][nt][j], sc[0][nt][j + 2]);
#pragma unroll
                for (int n = 1; n < EACH; ++n) mx[j] = max3(mx[j], sc[n][nt][j], sc[n][nt][j + 2]);
                mx[j] *= fit[nt][j];                                      // maxima live on the base-2 scale
                grown = grown || mx[j] > m[nt][j] + LAG;                  // (also for the first key a row sees)
            }
            if (__any_sync(0xffffffffu, grown)) {
#pragma unroll
                for (int j = 0; j < 2; ++j) {                             // over the keys: the lanes that share t
                    float top = mx[j];
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
                    const float m_new = top > m[nt][j] + LAG ? top : m[nt][j];        // (by this row alone, whatever the rows beside it)
                    const float shrink = m_new == -INFINITY ? 1.f : ex2(m[nt][j] - m_new);
                    m[nt][j] = m_new;
                    l[nt][j] *= shrink;
#pragma unroll
                    for (int d = 0; d < KSTEPS; ++d) {
                        o[nt][d][j] *= shrink;
                        o[nt][d][j + 2] *= shrink;
                    }
                }
            }
            float safe[2];
#pragma unroll
            for (int j = 0; j < 2; ++j) safe[j] = m[nt][j] == -INFINITY ? 0.f : m[nt][j] - BIAS;     // no key seen yet: keep exponents finite
#pragma unroll
            for (int n = 0; n < EACH; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    sc[n][nt][e] = ex2(fmaf(sc[n][nt][e], fit[nt][e & 1], -safe[e & 1]));
                    l[nt][e & 1] += sc[n][nt][e];
                }
#pragma unroll
            for (int n = 0; n < EACH; ++n)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    if (PARTS == 2) {
                        unsigned hi2, lo2;
                        split2(sc[n][nt][2 * h], sc[n][nt][2 * h + 1], hi2, lo2);
                        ph[n][nt][h] = movmatrix_trans(hi2);
                        pl[n][nt][h] = movmatrix_trans(lo2);
                    } else {
                        ph[n][nt][h] = movmatrix_trans(bits(__floats2half2_rn(sc[n][nt][2 * h], sc[n][nt][2 * h + 1])));
                    }
                }
        }
        // ---- values: tokens 2t, 2t + 1, 2t + 8, 2t + 9, coordinates HD / 8 * g and the next.  A token's numbers are words, the operand
        // wants a coordinate of two tokens side by side: the half bytes are exchanged before they are converted.
        constexpr int VW = HD / 64;                               // words of a token a lane has
#pragma unroll
        for (int n = 0; n < EACH; ++n) {
            const unsigned char* rec = vr + n * APART * RECORD;
            unsigned vw[4][VW], byte[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int key = 2 * t + (i & 1) + 8 * (i >> 1);
                const unsigned char* at = rec + key * (HD / 2) + g * (HD / 16);
                if (VW == 2) {
                    const uint2 v = *reinterpret_cast<const uint2*>(at);
                    vw[i][0] = v.x;
                    vw[i][VW - 1] = v.y;
                } else {
                    vw[i][0] = *reinterpret_cast<const unsigned*>(at);
                }
                byte[i] = rec[CODES + key * (HD / 16) + g * HD / 128];
            }
            if (!inside) {
                // (what lies outside the keys in use may be anything: its weight is zero, and so is made what it is multiplied by)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int kpos = k0 + n * STEP + 2 * t + (i & 1) + 8 * (i >> 1);
                    if (kpos < lo || kpos >= hi) byte[i] = 0;
                }
            }
            if (UNEVEN && !clear) {
                bool none = false;
#pragma unroll
                for (int i = 0; i < 4; ++i) none = none || byte[i] == FP4_NAN_SCALE;
                if (__any_sync(0xffffffffu, none)) hide_nan(p, byte, k0 + n * STEP);
            }
            __half2 vs[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const unsigned u = mad(byte[2 * i + 1], 1u << 23, mad(byte[2 * i], 1u << 7, 0u));
                vs[i] = *reinterpret_cast<const __half2*>(&u);
            }
#pragma unroll
            for (int w = 0; w < VW; ++w) {
                __half2 even[2][4], odd[2][4];                    // coordinates 2e and 2e + 1 of the word, of tokens 2i and 2i + 1
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const unsigned x = vw[2 * i][w], y = vw[2 * i + 1][w];
                    fp4_unpack(select_bits(0x0f0f0f0fu, x, mad(y, 16u, 0u)), even[i]);
                    fp4_unpack(select_bits(0x0f0f0f0fu, x >> 4, y), odd[i]);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        even[i][e] = __hmul2(even[i][e], vs[i]);
                        odd[i][e] = __hmul2(odd[i][e], vs[i]);
                    }
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int d = 4 * w + e;
                    const unsigned f[4] = {bits(even[0][e]), bits(odd[0][e]), bits(even[1][e]), bits(odd[1][e])};
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        if (PARTS == 2) {
                            float s[4] = {0.f, 0.f, 0.f, 0.f};
                            mma_f16(s, f, pl[n][nt][0], pl[n][nt][1]);
                            mma_f16(s, f, ph[n][nt][0], ph[n][nt][1]);
#pragma unroll
                            for (int x = 0; x < 4; ++x) o[nt][d][x] += s[x];
                        } else {
                            mma_f16(o[nt][d], f, ph[n][nt][0], ph[n][nt][1]);
                        }
                    }
                }
            }
        }
    }

    // Results of a warp that has rows of its own: into out, or a part's sums.  A lane's numbers of a row are neighbours.
    template <typename Row> __device__ __forceinline__ void finish(float* part, int part_rows, int row_in_part, int n_rows, Row out_row) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                float sum = l[nt][j];
                sum += __shfl_xor_sync(0xffffffffu, sum, 4);
                sum += __shfl_xor_sync(0xffffffffu, sum, 8);
                sum += __shfl_xor_sync(0xffffffffu, sum, 16);
                const int rr = nt * 8 + 2 * t + j;
                if (rr < n_rows) {
                    // (no sum: a row without a key.  Rows of a warp's own are float32: a query there that is not finite has a remainder that is no
                    // number, so that its sum is none either, also where every score is -inf)
                    const float inv = part != nullptr ? 1.f : sum == 0.f ? 0.f : 1.f / sum;
                    const int at = row_in_part + rr;
#pragma unroll
                    for (int d = 0; d < KSTEPS; d += 2) {
                        const float4 v = make_float4(o[nt][d][j] * inv, o[nt][d][j + 2] * inv, o[nt][d + 1][j] * inv, o[nt][d + 1][j + 2] * inv);
                        if (part != nullptr) __stcg(reinterpret_cast<float4*>(part + at * HD + g * (HD / 8) + 2 * d), v);
                        else store4(out_row(at) + g * (HD / 8) + 2 * d, v);
                    }
                    if (part != nullptr && g == 0)      // (no maximum remembers a score that is not a number)
                        __stcg(reinterpret_cast<float2*>(part + part_rows * HD + 2 * at), make_float2(sum != sum ? NAN : m[nt][j], sum));
                }
            }
    }

    // the warp's results: Om [NCW][rows][OPITCH], Mm and Lm [NCW][ROWS]
    __device__ __forceinline__ void leave(float* Om, float* Mm, float* Lm, int warp, int rows, int n_rows) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                float sum = l[nt][j];
                sum += __shfl_xor_sync(0xffffffffu, sum, 4);
                sum += __shfl_xor_sync(0xffffffffu, sum, 8);
                sum += __shfl_xor_sync(0xffffffffu, sum, 16);
                const int rr = nt * 8 + 2 * t + j;
                if (rr < n_rows) {
#pragma unroll
                    for (int d = 0; d < KSTEPS; ++d)
                        *reinterpret_cast<float2*>(Om + (warp * rows + rr) * OPITCH + g * (HD / 8) + 2 * d) = make_float2(o[nt][d][j], o[nt][d][j + 2]);
                    if (g == 0) {
                        Mm[warp * ROWS + rr] = sum != sum ? NAN : m[nt][j];     // (no maximum remembers a score that is not a number)
                        Lm[warp * ROWS + rr] = sum;
                    }
                }
            }
    }
};
// (a maximum that is not a number is kept: the row is not a number)
__device__ __forceinline__ float max_keep(float a, float b) { return (a != a || b != b) ? NAN : fmaxf(a, b); }

// OWN: every consumer warp has 8 NT rows of its own and takes all records of a tile; else the warps share the rows, and a tile's records.  UNEVEN: requests
// may bring several tokens, whose rows do not see the same keys (steps of single tokens are 1 to 4 % faster without what that takes:
// 8 requests of 2,049 12.0 us and 12.3, 4 of 27,001 to 32,767 36.8 and 38.3).
template <typename T, int HD, int STAGES, int NT, bool OWN, bool UNEVEN>
__global__ void __launch_bounds__(NTHREADS, (NT == 1 && sizeof(T) == 2) ? 3 : 2) attention_fp4_decode_kernel(const Params p) {
    using C = Consumer<T, HD, NT, UNEVEN>;
    constexpr int ROWS = (OWN ? NCW : 1) * 8 * NT, RECORD = fp4_record_bytes(HD);
    constexpr unsigned STAGE = 2 * RECORDS * RECORD;
    extern __shared__ __align__(128) unsigned char smem[];        // the ring, then the warps' results
    float* Om = reinterpret_cast<float*>(smem + STAGES * STAGE);
    __shared__ float Mm[OWN ? 1 : NCW * ROWS], Lm[OWN ? 1 : NCW * ROWS];
    __shared__ __align__(8) unsigned long long full_bar[STAGES];
    __shared__ __align__(8) unsigned long long empty_bar[STAGES];
    __shared__ int failed_flag, arrived, gave_up;

    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    if (tid == NCW * 32) {
        failed_flag = 0;
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(&full_bar[s], 1);
            mbar_init(&empty_bar[s], NCW);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    grid_launch_dependents();
    grid_dependency_wait();         // (lengths, tables and the cache itself may come from the kernels before this one)
    Walk w;
    if (!walk_first<ROWS>(p, w, lane)) return;          // (the same for all warps)
    __syncthreads();

    if (warp == NCW) {
        // ---- producer: lane = record of the tile (of keys, of values)
        asm volatile("fence.proxy.async.global;" ::: "memory");
        int it = 0, s = 0;
        unsigned phase = 1;                             // (a barrier that nobody has waited for yet lets the wait for parity 1 pass)
        bool ok = true;
        do {
            const int* table = p.block_table + (size_t)w.k.b * p.table_stride;
            for (int i = w.t0; i < w.t1; ++i, ++it) {
                if (!warp_wait(&empty_bar[s], phase, &failed_flag, p.status, ERR_PRODUCER_WAIT, lane)) {
                    ok = false;
                    break;
                }
                const int rec = (w.k.start + i * BN) / FP4_RECORD + (lane & (RECORDS - 1));
                const bool mine = lane < 2 * RECORDS && rec * FP4_RECORD < w.k.hi;
                const unsigned there = __ballot_sync(0xffffffffu, mine);
                if (lane == 0) mbar_expect_tx(&full_bar[s], __popc(there) * RECORD);
                __syncwarp();
                if (mine) {
                    const int block = p.page_shift >= 0 ? rec >> p.page_shift : rec / p.page_records;
                    long long page = table[block];
                    if (!tl_check_page(page) || page < 0 || page >= p.n_pages) page = 0;       // (a bad page is not followed; debug builds report it)
                    const long long at = ((page * p.n_kv_heads + w.kvh) * p.page_records + rec - block * p.page_records) * RECORD;
                    bulk_load(smem + s * STAGE + lane * RECORD, (lane < RECORDS ? p.k_pages : p.v_pages) + at, RECORD, &full_bar[s]);
                }
                __syncwarp();
                if (++s == STAGES) {
                    s = 0;
                    phase ^= 1u;
                }
            }
        } while (ok && walk_next<ROWS>(p, w));
        // (nothing that is still on its way may land in shared memory that is no longer this CTA's)
        int never = 0;
        for (int k = max(0, it - STAGES); k < it; ++k) mbar_wait(&full_bar[k % STAGES], (k / STAGES) & 1, &never);
        return;
    }

    // ---- consumers: all rows of the block and two records of every tile each, or rows of a warp's own and all records
    C c;
    bool ok = true;
    int s = 0;
    unsigned phase = 0;
    do {
        Block mine = w.k;
        if (OWN) {
            mine.row0 += warp * 8 * NT;
            mine.n_rows = min(max(mine.n_rows - warp * 8 * NT, 0), 8 * NT);
        }
        c.begin(p, mine, w.kvh, lane);
        for (int i = w.t0; i < w.t1; ++i) {
            if (!ok || !warp_wait(&full_bar[s], phase, &failed_flag, p.status, ERR_CONSUMER_WAIT, lane)) {
                ok = false;
                break;
            }
            const unsigned char* kr = smem + s * STAGE;
            if (OWN) {
#pragma unroll 1
                for (int r = 0; r < RECORDS; r += EACH)
                    c.template records<1>(p, kr + r * RECORD, kr + (RECORDS + r) * RECORD, w.k.start + i * BN + r * FP4_RECORD, w.k.lo, w.k.hi);
            } else {
                c.template records<NCW>(p, kr + warp * RECORD, kr + (RECORDS + warp) * RECORD, w.k.start + i * BN + warp * FP4_RECORD, w.k.lo, w.k.hi);
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&empty_bar[s]);     // this warp is done with the stage
            if (++s == STAGES) {
                s = 0;
                phase ^= 1u;
            }
        }
        if (UNEVEN) c.spoil();
        auto out_row = [&](int rr) {
            const int row = w.k.row0 + rr, token = token_of(p, row);
            return reinterpret_cast<T*>(p.out) + ((size_t)(w.k.first + token) * p.n_heads + w.kvh * p.group + row - token * p.group) * HD;
        };
        // what a row without a sum is multiplied by: zeros for one without a key; where all scores are -inf, from a query that is not finite, there is no softmax
        auto unsummed = [&](int rr) { return w.k.base + token_of(p, w.k.row0 + rr) >= 0 ? NAN : 0.f; };
        // where a part of this block lies: that with its first tile in its CTA's first place, others in the second
        const size_t place = part_floats(p.rows, HD);
        auto part_of = [&](int cta, bool first) { return p.part + ((size_t)cta * 2 + (first ? 0 : 1)) * place; };
        if (OWN && w.parts == 1) {
            if (ok) c.finish(nullptr, 0, warp * 8 * NT, mine.n_rows, out_row);
            continue;
        }
        // ---- the four warps' results, through shared memory
        consumers_sync();
        if (!OWN) c.leave(Om, Mm, Lm, warp, p.rows, w.k.n_rows);
        // (the producer may give up at any moment: one thread reads the flag for all, so that all take the same way
        // through the barriers below; what this part is made of has arrived by now, or a consumer has set the flag)
        if (tid == 0) gave_up = *(volatile int*)&failed_flag;
        consumers_sync();
        const bool sound = gave_up == 0;
        const int n_rows = w.k.n_rows;
        if (OWN) {
            if (sound) c.finish(part_of(blockIdx.x, w.t0 == 0), p.rows, warp * 8 * NT, mine.n_rows, out_row);
        } else if (sound) {
            float* part = part_of(blockIdx.x, w.t0 == 0);
            for (int idx = tid; idx < n_rows * (HD / 4); idx += NCW * 32) {      // four columns of a row per turn
                const int rr = idx / (HD / 4), d = (idx - rr * (HD / 4)) * 4;
                float M = -INFINITY, den = 0.f;
#pragma unroll
                for (int v = 0; v < NCW; ++v) M = max_keep(M, Mm[v * ROWS + rr]);
                float4 num = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                for (int v = 0; v < NCW; ++v) {
                    const float mv = Mm[v * ROWS + rr];
                    if (mv == -INFINITY) continue;
                    const float f = ex2(mv - M);
                    const float4 o4 = *reinterpret_cast<const float4*>(Om + (v * p.rows + rr) * C::OPITCH + d);
                    num.x = fmaf(f, o4.x, num.x); num.y = fmaf(f, o4.y, num.y);
                    num.z = fmaf(f, o4.z, num.z); num.w = fmaf(f, o4.w, num.w);
                    den = fmaf(f, Lm[v * ROWS + rr], den);
                }
                if (w.parts == 1) {
                    const float inv = M == -INFINITY ? unsummed(rr) : 1.f / den;
                    store4(out_row(rr) + d, make_float4(num.x * inv, num.y * inv, num.z * inv, num.w * inv));
                } else {
                    __stcg(reinterpret_cast<float4*>(part + rr * HD + d), num);
                    if (d == 0) __stcg(reinterpret_cast<float2*>(part + p.rows * HD + 2 * rr), make_float2(M, den));
                }
            }
        }
        // ---- whoever is last with a block's parts adds them up, in order
        if (w.parts > 1) {
            consumers_sync();
            int* counter = p.counters + ((size_t)w.k.b * p.blocks + w.k.number) * p.n_kv_heads + w.kvh;
            if (tid == 0) {
                // (release what the barrier has gathered of all threads' stores, acquire what the others released)
                const int add = sound ? 1 : 1 + FAILED_PART;
                int before;
                asm volatile("atom.add.acq_rel.gpu.global.s32 %0, [%1], %2;" : "=r"(before) : "l"(counter), "r"(add) : "memory");
                arrived = before + add;
                const int done = arrived & (FAILED_PART - 1);
                if (done >= w.parts) *counter = 0;
                if (done > w.parts) atomicExch(p.status, ERR_COUNT);      // (another call counts in the same place)
            }
            consumers_sync();
            if (arrived == w.parts) {
                // (eight parts at a time are under way)
                const int cta0 = (w.off + worth_of(ROWS)) / w.share;
                for (int idx = tid; idx < n_rows * (HD / 4); idx += NCW * 32) {
                    const int rr = idx / (HD / 4), d = (idx - rr * (HD / 4)) * 4;
                    float4 num = make_float4(0.f, 0.f, 0.f, 0.f);
                    float M = -INFINITY, den = 0.f;
                    for (int c0 = 0; c0 < w.parts; c0 += 8) {
                        float2 ml[8];
                        float4 o4[8];
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            ml[i] = make_float2(-INFINITY, 0.f);
                            o4[i] = make_float4(0.f, 0.f, 0.f, 0.f);
                            if (c0 + i < w.parts) {
                                const float* part = part_of(cta0 + c0 + i, c0 + i == 0);
                                ml[i] = __ldcg(reinterpret_cast<const float2*>(part + p.rows * HD + 2 * rr));
                                o4[i] = __ldcg(reinterpret_cast<const float4*>(part + rr * HD + d));
                            }
                        }
                        float top = M;
#pragma unroll
                        for (int i = 0; i < 8; ++i) top = max_keep(top, ml[i].x);
                        const float old = M == -INFINITY ? 0.f : ex2(M - top);
                        num.x *= old; num.y *= old; num.z *= old; num.w *= old;
                        den *= old;
                        M = top;
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            if (ml[i].x == -INFINITY) continue;
                            const float f = ex2(ml[i].x - M);
                            num.x = fmaf(f, o4[i].x, num.x); num.y = fmaf(f, o4[i].y, num.y);
                            num.z = fmaf(f, o4[i].z, num.z); num.w = fmaf(f, o4[i].w, num.w);
                            den = fmaf(f, ml[i].y, den);
                        }
                    }
                    const float inv = M == -INFINITY ? unsummed(rr) : 1.f / den;
                    store4(out_row(rr) + d, make_float4(num.x * inv, num.y * inv, num.z * inv, num.w * inv));
                }
            }
        }
        consumers_sync();            // the place behind the stages is the next part's
    } while (walk_next<ROWS>(p, w));
}

// ---- host side ---------------------------------------------------------------------------------

template <int HD> constexpr int stages_for() { return HD == 128 ? 3 : 5; }
template <int HD> size_t smem_for(int rows, bool own) {
    return (size_t)stages_for<HD>() * 2 * RECORDS * fp4_record_bytes(HD) + (own ? 0 : (size_t)NCW * rows * (HD + 4) * 4);
}

bool takes(int n_heads, int n_kv_heads, int head_dim, int page_size) {
    if (head_dim != 64 && head_dim != 128) return false;
    if (n_heads <= 0 || n_kv_heads <= 0 || n_heads % n_kv_heads != 0) return false;
    return page_size >= FP4_RECORD && page_size % FP4_RECORD == 0;
}

struct Plan {
    bool own, uneven;
    int nt, rows, blocks, ctas;
    size_t smem;
};

template <typename T, int HD, int NT, bool OWN, bool UNEVEN> int ctas_per_sm(int rows) {
    static int known[8 * NT * NCW + 1] = {};               // (threads that come here at the same time write the same)
    if (known[rows] == 0) {
        auto kern = attention_fp4_decode_kernel<T, HD, stages_for<HD>(), NT, OWN, UNEVEN>;
        int n = 0;
        if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem_for<HD>(8 * NT, OWN)) != cudaSuccess ||
            cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kern, NTHREADS, smem_for<HD>(rows, OWN)) != cudaSuccess || n < 1) {
            cudaGetLastError();
            n = 1;
        }
        known[rows] = n;
    }
    return known[rows];
}
template <typename T, int HD, bool UNEVEN> int ctas_per_sm(int nt, int rows) {
    return nt == 1 ? ctas_per_sm<T, HD, 1, false, UNEVEN>(rows) : ctas_per_sm<T, HD, 2, false, UNEVEN>(rows);
}
template <int HD> int ctas_per_sm(int dtype, const Plan& pl) {
    if (pl.own) return ctas_per_sm<float, HD, 2, true, true>(pl.rows);
    if (dtype == TL_F32) return pl.uneven ? ctas_per_sm<float, HD, true>(pl.nt, pl.rows) : ctas_per_sm<float, HD, false>(pl.nt, pl.rows);
    return pl.uneven ? ctas_per_sm<__nv_bfloat16, HD, true>(pl.nt, pl.rows) : ctas_per_sm<__nv_bfloat16, HD, false>(pl.nt, pl.rows);
}

Plan make_plan(int dtype, int n_seqs, int n_heads, int n_kv_heads, int head_dim, int max_q_len, int max_kv_len) {
    Plan pl;
    const long long all = (long long)max_q_len * (n_heads / n_kv_heads);
    // float32 steps of many rows: rows of its own for each warp, where that gives 96 blocks or more.  (us, shared rows and own: 32 / 8 heads of 64,
    // 3 requests of 64 tokens behind 500, 96 blocks, 24.1 25.5; one of 128, 64 blocks, 19.4 25.5; one of 512, 256 blocks, 54.6 50.1; 8 of 512 behind 4,000
    // 1,430 1,210; heads of 128: 52.6 46.3; 39.4 45.9; 136 94; 4,167 2,333.)
    constexpr int OWN = NCW * 16;
    pl.own = dtype == TL_F32 && all >= OWN && (double)n_seqs * ((all + OWN - 1) / OWN) * n_kv_heads >= 96.0;
    pl.uneven = max_q_len > 1;
    pl.nt = all <= 8 ? 1 : 2;
    const int most = 8 * pl.nt * (pl.own ? NCW : 1);
    pl.rows = all < most ? (int)all : most;
    pl.blocks = (int)((all + most - 1) / most);
    pl.smem = head_dim == 128 ? smem_for<128>(pl.rows, pl.own) : smem_for<64>(pl.rows, pl.own);
    const int fit = head_dim == 128 ? ctas_per_sm<128>(dtype, pl) : ctas_per_sm<64>(dtype, pl);
    // no more CTAs than there can be tiles
    const double tiles = (double)n_seqs * pl.blocks * n_kv_heads * ((max_kv_len + BN - 1) / BN + 1);
    pl.ctas = tiles < (double)SMS * fit ? (int)tiles : SMS * fit;
    if (pl.ctas < 1) pl.ctas = 1;
    return pl;
}

// (ctas_per_sm has raised the limit on shared memory)
template <typename T, int HD, int NT, bool OWN, bool UNEVEN> int launch(const Params& p, const Plan& pl, cudaStream_t s) {
    return (int)tl_launch(attention_fp4_decode_kernel<T, HD, stages_for<HD>(), NT, OWN, UNEVEN>, dim3(pl.ctas), dim3(NTHREADS), pl.smem, s, p);
}
template <typename T, int HD, bool UNEVEN> int launch(const Params& p, const Plan& pl, cudaStream_t s) {
    return pl.nt == 1 ? launch<T, HD, 1, false, UNEVEN>(p, pl, s) : launch<T, HD, 2, false, UNEVEN>(p, pl, s);
}
template <int HD> int launch(int dtype, const Params& p, const Plan& pl, cudaStream_t s) {
    if (pl.own) return launch<float, HD, 2, true, true>(p, pl, s);
    if (dtype == TL_F32) return pl.uneven ? launch<float, HD, true>(p, pl, s) : launch<float, HD, false>(p, pl, s);
    return pl.uneven ? launch<__nv_bfloat16, HD, true>(p, pl, s) : launch<__nv_bfloat16, HD, false>(p, pl, s);
}

}  // namespace

// What a call needs beside its operands: workspace_floats of scratch, and n_counters ints that are zero (and are zero again when
// the call has run); no call that may run at the same time may have either.
extern "C" int tl_attention_fp4_decode_plan(int dtype, int n_seqs, int n_heads, int n_kv_heads, int head_dim, int page_size, int max_q_len,
                                            int max_kv_len, long long* workspace_floats, long long* n_counters) {
    if (!takes(n_heads, n_kv_heads, head_dim, page_size) || max_q_len < 1 || n_seqs < 1) return TL_BAD_SIZE;
    if (dtype != TL_BF16 && dtype != TL_F32) return TL_BAD_DTYPE;
    const Plan pl = make_plan(dtype, n_seqs, n_heads, n_kv_heads, head_dim, max_q_len, max_kv_len);
    *workspace_floats = (long long)pl.ctas * 2 * part_floats(pl.rows, head_dim);
    *n_counters = (long long)n_seqs * pl.blocks * n_kv_heads;
    return TL_OK;
}

// q, out: [tokens, n_heads, head_dim] of dtype; pages: [n_pages, n_kv_heads, page_size / 16, 9 head_dim] bytes; block_table: [n_seqs,
// table_cols] with rows table_stride apart; q_start may count from anywhere in q.
extern "C" int tl_attention_fp4_decode(const void* q, const void* k_pages, const void* v_pages, void* out, const int* block_table,
                                       int table_stride, int table_cols, const int* q_start, const int* kv_len, float* workspace,
                                       int* counters, int* status, int dtype, int n_seqs, int n_heads, int n_kv_heads, int head_dim,
                                       int page_size, long long n_pages, int max_q_len, int max_kv_len, int window, float scale, void* stream) {
    if (n_seqs <= 0 || max_q_len <= 0) return TL_OK;
    if (!takes(n_heads, n_kv_heads, head_dim, page_size) || n_pages <= 0 || max_kv_len < 0 || !fp4_places_fit(table_cols, page_size, max_q_len)) return TL_BAD_SIZE;
    if (dtype != TL_BF16 && dtype != TL_F32) return TL_BAD_DTYPE;
    if (!aligned16(q) || !aligned16(out) || !aligned16(k_pages) || !aligned16(v_pages) || !aligned16(workspace)) return TL_BAD_ALIGN;
    if (workspace == nullptr || counters == nullptr || status == nullptr) return TL_BAD_SIZE;
    const Plan pl = make_plan(dtype, n_seqs, n_heads, n_kv_heads, head_dim, max_q_len, max_kv_len);
    if ((double)n_seqs * pl.blocks * n_kv_heads * ((double)table_cols * page_size / BN + 3) >= 2147483647.0) return TL_BAD_SIZE;
    Params p;
    p.q = q; p.out = out; p.k_pages = (const unsigned char*)k_pages; p.v_pages = (const unsigned char*)v_pages;
    p.block_table = block_table; p.q_start = q_start; p.kv_len = kv_len;
    p.part = workspace; p.counters = counters; p.status = status; p.n_pages = n_pages;
    p.table_stride = table_stride; p.table_cols = table_cols; p.n_seqs = n_seqs; p.n_heads = n_heads; p.n_kv_heads = n_kv_heads;
    p.group = n_heads / n_kv_heads; p.page_records = page_size / FP4_RECORD; p.blocks = pl.blocks; p.rows = pl.rows;
    p.page_shift = -1;
    for (int b = 0; b < 31; ++b)
        if (p.page_records == 1 << b) p.page_shift = b;
    p.per_group = p.group == 1 ? 0u : (unsigned)((1ull << 32) / (unsigned)p.group) + 1u;
    if ((double)max_q_len * p.group * p.group >= 4294967296.0) return TL_BAD_SIZE;
    p.window = fp4_window(window, table_cols, page_size);
    p.scale_log2 = scale * LOG2E;
    cudaStream_t s = (cudaStream_t)stream;
    return head_dim == 128 ? launch<128>(dtype, p, pl, s) : launch<64>(dtype, p, pl, s);
}
