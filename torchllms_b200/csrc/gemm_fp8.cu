// C[m, n] = sum_kb sx[m, kb] sw[n, kb] sum_{k in block kb} x[m, k] w[n, k]: products of 8-bit rows with 8-bit weights (format:
// fp8.cuh) on the fifth-generation tensor cores, any number of rows; and the same for routed experts, whose rows stand
// sorted by expert.
//
// The scales are powers of two, one for 128 numbers, which is what the block-scaled instruction (kind::mxf8f6f4, E8M0 scales in
// tensor memory) multiplies by: no sum has to leave tensor memory between blocks, and every product and its scaling is exact
// in float32.  The instruction takes a scale for 32 numbers; here four instructions in a row are told the same byte.
//
// The operands are swapped as in gemm_tcgen05.cu: rows of W are the M of the instruction (128 a CTA), rows of x its N (`width`,
// up to 240, chosen per call, so that few rows waste little).  D[w_row, token] lies with a row of W to a TMEM lane.
//
// Three forms, by a rule on sizes at the end of this file:
//   single  a persistent CTA per SM walks units (a slab of 128 rows of W, a tile of rows of x), tiles fastest, so that a slab of W comes
//           from memory once and the rows of x, which are fewer, from L2;
//   pairs   the same by two CTAs that share a unit of 256 rows of W (cta_group::2): each brings its half of the tile's rows of x;
//   split   few units: the blocks of K of each are dealt out to the CTAs of a cluster, whose sums meet through distributed shared memory
//           and are added up in the order of K.
// And three ends: the sums leave (float32 or bfloat16), or 8-bit rows of act(sum) do, or of act(gate) * up.
//
// Inside a CTA:
//   warp 0     TMA: boxes of W [128 x 128] and of x [width x 128], 128-byte swizzle, one or two of each a stage; the first ones of W are asked
//              for into L2 before the kernel ahead of this one has ended
//   warp 1     tcgen05.cp of scales (a word a row: four blocks of 128) and tcgen05.mma, four of K 32 a box; by one lane, as warp 0's loads
//              (64 rows of 4,096 x 14,336 by pairs: 34.2 us with the lane elected at each instruction, 24.6 so, 21.9 with warp 0 so too)
//   warps 2, 3 scales from memory to shared memory, four words a row and turn (2,048 of K), in turns; in the order that tcgen05.cp
//              wants: row r of a chunk of 128 at 16 (r % 32) + 4 (r / 32).  (The fence behind them waits for all loads under way: a
//              word a turn, copied ahead, kept the products waiting, 49 us for 39 in the same case and 225 for 203 with 2,048 rows of 28,672 x 4,096.)
//   the rest   results: tcgen05.ld, through shared memory to rows of C; two accumulators, so that the next unit's products run meanwhile
//
// Measured (microseconds of repeated calls; floors at 6.57 TB/s and twice the 16-bit rate of 1.65 PFLOP/s): 8 rows of 28,672 x 4,096 22.9 (floor
// 18.1: 224 slabs on 148 SMs, one or two each), 64 of 4,096 x 14,336 15.8 (9.2), 2,048 of 28,672 x 4,096 208 to 217 under the power cap that
// long runs of it meet, 172 to 181 in short ones (146; 122 is what the tensor pipe is busy for).  What bounds the last, from copies of an
// earlier step (203 us in short runs) with a part left out: no copies of scales 168, no loads 158, one product in four 126, no products 105.
// Every wait is bounded: on a time-out the CTA records a code, lets its copies land, frees its tensor memory and returns.
#include "fp8.cuh"
#include <cuda.h>

namespace {

constexpr int BM = 128;              // rows of W a CTA
constexpr int BK = 128;              // bytes of K a box: a swizzle row, and a block of numbers that share a scale
constexpr int MAX_WIDTH = 240;       // rows of x a tile: two accumulators and two sets of scales fill 512 columns
// Split: tiles so narrow send their sums to where they are added up, wider ones, whose sums would take room from the stages, leave them to
// be fetched (8 rows of 4,096 x 14,336: 13.5 us sent, 14.6 fetched; 64 rows 15.9 and 15.7); and tiles so narrow share an SM.
constexpr int PUSH_WIDTH = 32;
constexpr int SHARED_WIDTH = 64;
constexpr int MAX_SPLIT_WIDTH = 224; // the same with one accumulator in 256 columns
constexpr int COLUMNS = 256;
constexpr int MAX_STAGES = 12;
constexpr int MAX_SCALE_BUFS = 3;    // turns of scales under way
constexpr int TURN = 16;             // blocks of 128 of a turn: four words a row
enum : int { SINGLE = 1, PAIRS = 2, SPLIT = 3 };
enum : int { PLAIN = 0, ACT = 1, GATED = 2 };       // what becomes of the sums: they leave; 8-bit rows of act(sum); of act(gate) * up
// Warps that take the results: eight, two to a quarter of tensor memory's lanes, with every other 32 columns each (one warp a scheduler
// waits for its own instructions: 524 us for 275 where 2,048 tokens go through gates and ups of 32 experts); split, four, where
// two CTAs share an SM.
__host__ __device__ constexpr int result_warps(int form) { return form == SPLIT ? 4 : 8; }       // (two CTAs of SPLIT may share an SM)
__host__ __device__ constexpr int threads_of(int form) { return 32 * (4 + result_warps(form)); }
constexpr int STAGING = 8 * 2048;    // 32 x 32 results a warp
constexpr unsigned ACC_COLS = 256;   // a second accumulator lies so many columns behind the first
constexpr unsigned long long WAIT_LIMIT_NS = 2000ull * 1000ull * 1000ull;   // two seconds, then give up

enum : int { ERR_TMA_WAIT = 601, ERR_MMA_WAIT = 602, ERR_SCALE_WAIT = 603, ERR_EPI_WAIT = 604 };

__device__ __forceinline__ unsigned smem_u32(const void* p) { return (unsigned)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void mbar_init(unsigned bar, unsigned count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count));
}
// OTHERS: the waiting thread itself reads what another CTA of the cluster has stored here, so the wait acquires at the cluster's scope.  What the
// other waits guard is read by the tensor cores and the copy engine, or from tensor memory (an acquire at the cluster's scope in all of
// them took 8 rows of 28,672 x 4,096 from 34.7 us to 35.9).
template <bool OTHERS>
__device__ __forceinline__ bool mbar_try_wait(unsigned bar, unsigned parity) {
    unsigned ok;
    if (OTHERS)
        asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                     : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
    else asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                      : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
    return ok != 0;
}
__device__ __forceinline__ unsigned long long global_ns() {
    unsigned long long t;
    asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t));
    return t;
}
// false once the limit has passed, or as soon as another role has given up
template <bool OTHERS = false>
__device__ __forceinline__ bool wait_one(unsigned bar, unsigned parity, volatile int* aborted) {
    bool ok = mbar_try_wait<OTHERS>(bar, parity);
    unsigned long long t0 = 0;
    // (the timer is read rarely: a read takes as long as a stage's products)
    for (unsigned i = 1; !ok; ++i) {
        ok = mbar_try_wait<OTHERS>(bar, parity);
        if (!ok && (i & 255u) == 0u) {
            if (t0 == 0) t0 = global_ns();
            if (*aborted || global_ns() - t0 > WAIT_LIMIT_NS) break;
        }
    }
    return ok;
}
// the same for a whole warp that waits together
template <bool OTHERS = false>
__device__ __forceinline__ bool mbar_wait(unsigned bar, unsigned parity, volatile int* aborted) {
    return __all_sync(0xffffffffu, wait_one<OTHERS>(bar, parity, aborted));
}
__device__ __forceinline__ void give_up(volatile int* aborted, int* status, int code) {
    *aborted = 1;
    atomicExch(status, code);
}
// One elected lane of a warp in step arrives.  PAIR: at a barrier that may be the other CTA's.  (Neither form orders more than this CTA
// sees: what it guards has gone through a proxy fence or has been read from tensor memory.  Release at the cluster's scope, which waits for
// everything the warp has stored, took 8 rows of 28,672 x 4,096 from 31.2 us to 34.7.)
template <bool PAIR>
__device__ __forceinline__ void arrive_elect(unsigned bar) {
    if (!PAIR) {
        asm volatile("{\n\t.reg .pred e;\n\telect.sync _|e, 0xffffffff;\n\t@e mbarrier.arrive.shared::cta.b64 _, [%0];\n\t}" ::"r"(bar) : "memory");
        return;
    }
    asm volatile("{\n\t.reg .pred e;\n\telect.sync _|e, 0xffffffff;\n\t@e mbarrier.arrive.shared::cluster.b64 _, [%0];\n\t}" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// a word into another CTA's shared memory, counted by the barrier of the same place there
__device__ __forceinline__ void store_async(unsigned addr, unsigned v, unsigned bar, int cta) {
    unsigned at, there;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(addr), "r"(cta));
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(bar), "r"(cta));
    asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.b32 [%0], %1, [%2];" ::"r"(at), "r"(v), "r"(there) : "memory");
}
__device__ __forceinline__ void store_async4(unsigned at, const unsigned* v, unsigned bar) {
    asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.v4.b32 [%0], {%1, %2, %3, %4}, [%5];"
                 ::"r"(at), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(bar) : "memory");
}
// 16 bytes of another CTA's shared memory
__device__ __forceinline__ float4 load_from(unsigned addr, int cta) {
    unsigned at;
    float4 v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(addr), "r"(cta));
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(at) : "memory");
    return v;
}
// the address of another CTA's variable of the same place
__device__ __forceinline__ unsigned in_cta(unsigned addr, int cta) {
    unsigned r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(cta));
    return r;
}
__device__ __forceinline__ void expect_tx(unsigned bar, unsigned bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
// A box of x, or of W with a mark on what becomes of it in L2.  PAIR: the barrier that counts the bytes is the first CTA's.
template <bool PAIR>
__device__ __forceinline__ void tma_load(unsigned dst, const CUtensorMap* map, unsigned bar, int x, int y, unsigned long long policy) {
#define TL_LOAD(G) \
    asm volatile("cp.async.bulk.tensor.2d" G ".shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1, {%3, %4}], [%2], %5;" \
                 ::"r"(dst), "l"(map), "r"(bar), "r"(x), "r"(y), "l"(policy) : "memory")
    if (PAIR) TL_LOAD(".cta_group::2");
    else TL_LOAD("");
#undef TL_LOAD
}
// a box of a gated weight: 16 rows of gates and the 16 matching rows of ups in turn, four times
template <bool PAIR>
__device__ __forceinline__ void tma_load_gated(unsigned dst, const CUtensorMap* map, unsigned bar, int x, int group, int expert, unsigned long long policy) {
    const int zero = 0;
#define TL_LOAD(G) \
    asm volatile("cp.async.bulk.tensor.5d" G ".shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1, {%3, %4, %4, %5, %6}], [%2], %7;" \
                 ::"r"(dst), "l"(map), "r"(bar), "r"(x), "r"(zero), "r"(group), "r"(expert), "l"(policy) : "memory")
    if (PAIR) TL_LOAD(".cta_group::2");
    else TL_LOAD("");
#undef TL_LOAD
}
// The same boxes into L2 only.  L2 is where all writes to memory meet, so what a kernel that still runs writes later is read all the same.
__device__ __forceinline__ void prefetch_box(const CUtensorMap* map, int x, int y) {
    asm volatile("cp.async.bulk.prefetch.tensor.2d.L2.global.tile [%0, {%1, %2}];" ::"l"(map), "r"(x), "r"(y) : "memory");
}
__device__ __forceinline__ void prefetch_box_gated(const CUtensorMap* map, int x, int group) {
    const int zero = 0;
    asm volatile("cp.async.bulk.prefetch.tensor.5d.L2.global.tile [%0, {%1, %2, %2, %3, %2}];" ::"l"(map), "r"(x), "r"(zero), "r"(group) : "memory");
}
__device__ __forceinline__ void prefetch_line(const void* p) { asm volatile("prefetch.global.L2 [%0];" ::"l"(p)); }
__device__ __forceinline__ unsigned long long policy_first() {
    unsigned long long p;
    asm volatile("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(p));
    return p;
}
__device__ __forceinline__ unsigned long long policy_normal() {
    unsigned long long p;
    asm volatile("createpolicy.fractional.L2::evict_normal.b64 %0, 1.0;" : "=l"(p));
    return p;
}

// shared-memory matrix descriptors.  Operands: K-major, rows of 128 bytes, 128-byte swizzle, groups of 8 rows 1,024 bytes
// apart.  Scales: no swizzle, rows of 16 bytes, groups of 8 rows 128 bytes apart.
__device__ __forceinline__ unsigned long long operand_desc(unsigned addr) {
    return (unsigned long long)((addr & 0x3FFFFu) >> 4) | ((unsigned long long)(1024u >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
__device__ __forceinline__ unsigned long long scale_desc(unsigned addr) {
    return (unsigned long long)((addr & 0x3FFFFu) >> 4) | ((unsigned long long)(128u >> 4) << 32) | (1ull << 46);
}
// instruction descriptor: E4M3 x E4M3 with E8M0 scales, both K-major, M rows and N columns; the byte of the scales' words
__device__ __forceinline__ unsigned instruction(int M, int N, int byte) {
    return (1u << 23) | ((unsigned)(N >> 3) << 17) | ((unsigned)(M >> 4) << 24) | ((unsigned)byte << 29) | ((unsigned)byte << 4);
}
__device__ __forceinline__ bool elect_one() {
    unsigned e;
    asm volatile("{\n\t.reg .pred e;\n\telect.sync _|e, 0xffffffff;\n\tselp.u32 %0, 1, 0, e;\n\t}" : "=r"(e));
    return e != 0;
}
// One lane issues, always the same.  PAIR: for both CTAs, the first one issues; commits arrive at both CTAs' barriers.
template <bool PAIR>
__device__ __forceinline__ void mma(unsigned d, unsigned long long a, unsigned long long b, unsigned idesc, unsigned sa, unsigned sb, unsigned accumulate) {
#define TL_MMA(G) \
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t" \
                 "tcgen05.mma.cta_group::" #G ".kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" \
                 ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(sa), "r"(sb), "r"(accumulate) : "memory")
    if (PAIR) TL_MMA(2);
    else TL_MMA(1);
#undef TL_MMA
}
template <bool PAIR>
__device__ __forceinline__ void copy_scales(unsigned taddr, unsigned long long desc) {
#define TL_COPY(G) \
    asm volatile("tcgen05.cp.cta_group::" #G ".32x128b.warpx4 [%0], %1;" \
                 ::"r"(taddr), "l"(desc) : "memory")
    if (PAIR) TL_COPY(2);
    else TL_COPY(1);
#undef TL_COPY
}
template <bool PAIR>
__device__ __forceinline__ void commit(unsigned bar, unsigned short both) {
    if (PAIR)
        asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar), "h"(both) : "memory");
    else
        asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void tmem_load32(unsigned taddr, unsigned (&r)[32]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
                 "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
                   "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]),
                   "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]),
                   "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
                 : "r"(taddr));
}
__device__ __forceinline__ void tmem_load16(unsigned taddr, unsigned (&r)[16]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
                   "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
                 : "r"(taddr));
}
__device__ __forceinline__ void tmem_store16(unsigned taddr, const float (&v)[16]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
                 ::"r"(taddr), "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]), "f"(v[8]), "f"(v[9]),
                   "f"(v[10]), "f"(v[11]), "f"(v[12]), "f"(v[13]), "f"(v[14]), "f"(v[15]) : "memory");
}
// the result warps' barrier, which also tells whether all of them came through
__device__ __forceinline__ bool meet(bool ok) {
    unsigned all;
    __syncwarp();
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 q, %1, 0;\n\tbar.red.and.pred p, 1, 256, q;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                 : "=r"(all) : "r"((unsigned)ok) : "memory");
    return all != 0;
}
// The largest magnitude over LANES neighbouring lanes of each of their LANES values (bits of finite numbers): a lane is left with
// that of value number lane % LANES.  Each step halves the values and doubles the lanes that they stand for.
template <int LANES>
__device__ __forceinline__ unsigned largest_of_lanes(unsigned (&m)[LANES]) {
    const unsigned lane = threadIdx.x & 31;
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) {
        const bool high = lane & o;
#pragma unroll
        for (int j = 0; j < o; ++j) {
            const unsigned other = __shfl_xor_sync(0xffffffffu, high ? m[j] : m[j + o], o);
            m[j] = max(high ? m[j + o] : m[j], other);
        }
    }
    return m[0];
}
// up to four words of a row's scales, zeros where there is no row (null)
__device__ __forceinline__ void load_words(const unsigned char* at, int words, bool whole, unsigned (&v)[4]) {
    if (at != nullptr && whole) {        // (every turn of every row starts on 16 bytes and has 16)
        const uint4 r = *reinterpret_cast<const uint4*>(at);
        v[0] = r.x; v[1] = r.y; v[2] = r.z; v[3] = r.w;
        return;
    }
#pragma unroll
    for (int w = 0; w < 4; ++w) v[w] = at != nullptr && w < words ? *reinterpret_cast<const unsigned*>(at + 4 * w) : 0u;
}

struct Params {
    void* out;                       // [M, N] (experts: rows in sorted order)
    int* status;
    const unsigned char* w_scales;   // [experts * N][pitch]
    const unsigned char* x_scales;   // [M][pitch]
    const int* tiles;                // experts: count, then (expert, first row, rows) of every tile; null: one weight, tiles of `width` rows
    int M, N, k_blocks, pitch;
    int width;                       // rows of x a tile, a multiple of 16
    int slabs, n_tiles, stages, scale_bufs;
    int x_box;                       // rows of a box of x
    int out_is_f32;
    bool w_whole, x_whole;           // scales: rows are a multiple of 16 bytes and start on 16
    int push_bytes;                  // SPLIT, narrow tiles: where the CTAs of a cluster send what this one adds up
    int splits, split_blocks;        // SPLIT: CTAs of a cluster, and blocks of K of each (a multiple of 4)
    // ACT, GATED: the 8-bit rows that leave, [M, N] (GATED: [M, N / 2]), and what is done to the sums
    unsigned char *codes, *scales;
    int hidden;
    Fp8Gate gate;
    unsigned tmem_cols, scale_col, set_cols;     // columns of tensor memory; where the first set of scales lies, and how far the second is behind it
};

// shared memory of a word of scales: 512 bytes for the rows of W and for every 128 rows of x
__host__ __device__ constexpr int scale_bytes(int width) { return 512 * (1 + (width + 127) / 128); }

// Boxes of W (and of x) a stage.  Narrow tiles: two, what a stage costs its issuer (a wait, a fence, a commit) is more than its products
// take.  Wide ones, whose boxes are large: one, for the more even stream (2,048 tokens through gates and ups of 32 experts: 303 us
// and 249).  Split: one, the few blocks of a CTA would be a stage or two otherwise.
__host__ __device__ constexpr int boxes_of(int form) { return form == SINGLE ? 2 : 1; }

struct Unit { int expert, row0, rows, slab; };

__device__ __forceinline__ Unit unit_of(const Params& p, int u, int n_tiles) {
    Unit r;
    const int t = u % n_tiles;
    r.slab = u / n_tiles;
    if (p.tiles != nullptr) {
        r.expert = p.tiles[1 + 3 * t];
        r.row0 = p.tiles[2 + 3 * t];
        r.rows = p.tiles[3 + 3 * t];
    } else {
        r.expert = 0;
        r.row0 = t * p.width;
        r.rows = min(p.width, p.M - r.row0);
    }
    return r;
}

// SPLIT: groups of four rows of x are dealt out to the CTAs of a cluster: how many of a tile's one adds up
__device__ __forceinline__ int groups_of(int rows, int cta, int ctas) {
    const int groups = (rows + 3) / 4;
    return groups > cta ? (groups - cta - 1) / ctas + 1 : 0;
}

template <int FORM, int EPI, int ACTIVATION>
__global__ void __launch_bounds__(threads_of(FORM), FORM == SPLIT ? 2 : 1) gemm_fp8_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x,
                                                               const Params p) {
    extern __shared__ unsigned char smem_raw[];
    const unsigned smem0 = (smem_u32(smem_raw) + 1023u) & ~1023u;            // tiles want 1,024-byte alignment for the swizzle
    unsigned char* const smem_at = smem_raw + (smem0 - smem_u32(smem_raw));
    // a pair shares a unit of 256 rows of W: each CTA has 128 of them and half of the tile's rows of x
    constexpr bool PAIR = FORM == PAIRS, CUT = FORM == SPLIT;
    constexpr int BOXES = boxes_of(FORM);
    constexpr int SIDES = PAIR ? 2 : 1;
    const int rank = PAIR ? (int)(blockIdx.x & 1) : 0;
    // split: a cluster to a unit, every CTA with a run of its blocks of K
    const int group = (int)blockIdx.x / SIDES, cut = CUT ? group % p.splits : 0;
    const int first_unit = CUT ? group / p.splits : group;
    const int step = CUT ? p.n_tiles * p.slabs : (int)gridDim.x / SIDES;
    const int kb0 = cut * p.split_blocks, kb1 = CUT ? min(kb0 + p.split_blocks, p.k_blocks) : p.k_blocks;
    const unsigned w_bytes = BM * BK, x_bytes = p.width / SIDES * BK, stage_bytes = BOXES * (w_bytes + x_bytes);
    const unsigned scales_at = smem0 + p.stages * stage_bytes, word_bytes = scale_bytes(p.width), turn_bytes = 4 * word_bytes;
    unsigned char* const staging = smem_at + p.stages * stage_bytes + p.scale_bufs * turn_bytes;
    // ACT, GATED: a tile's largest magnitudes, by result warp; the other CTA's, of two units; what a row is multiplied by (a tile's
    // columns are taken 32 at a time: room for whole ones)
    unsigned* const tops = reinterpret_cast<unsigned*>(staging + STAGING);            // [4][COLUMNS]
    unsigned* const theirs = tops + 4 * COLUMNS;                                      // [2][COLUMNS]
    float* const inverse = reinterpret_cast<float*>(theirs + 2 * COLUMNS);            // [COLUMNS]
    __shared__ __align__(8) unsigned long long bars[2 * MAX_STAGES + 2 * MAX_SCALE_BUFS + 7];
    __shared__ unsigned tmem_slot;
    __shared__ int abort_flag;
    unsigned char* const pushed = staging;               // SPLIT (which stages nothing): [group of four rows of x of this CTA's][split][row of W][4]
    const unsigned bar0 = smem_u32(bars);
    const unsigned full = bar0, empty = bar0 + 8 * MAX_STAGES, sc_full = bar0 + 16 * MAX_STAGES, sc_empty = sc_full + 8 * MAX_SCALE_BUFS;
    const unsigned acc_full = sc_empty + 8 * MAX_SCALE_BUFS, acc_empty = acc_full + 16, drained = acc_empty + 16, told = drained + 8;
    // (what the first CTA's issuing warp waits for counts arrivals of both)
    auto leader = [&](unsigned bar) { return PAIR ? in_cta(bar, 0) : bar; };

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 32) {           // (descriptors come from memory: on their way while the barriers are set up)
        asm volatile("prefetch.tensormap [%0];" ::"l"(&map_w) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&map_x) : "memory");
    }
    if (threadIdx.x == 0) {
        abort_flag = 0;
        for (int s = 0; s < MAX_STAGES; ++s) { mbar_init(full + 8 * s, 1); mbar_init(empty + 8 * s, 1); }
        for (int s = 0; s < MAX_SCALE_BUFS; ++s) { mbar_init(sc_full + 8 * s, SIDES); mbar_init(sc_empty + 8 * s, 1); }
        for (int s = 0; s < 2; ++s) { mbar_init(acc_full + 8 * s, 1); mbar_init(acc_empty + 8 * s, result_warps(FORM) * SIDES); }
        mbar_init(drained, 1);
        if (EPI == GATED || CUT) { mbar_init(told, 1); mbar_init(told + 8, 1); }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        if (PAIR) {
            asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)), "r"(p.tmem_cols) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
        } else {
            asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)), "r"(p.tmem_cols) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        }
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (PAIR) cluster_sync();          // both CTAs' barriers are set up and both have their tensor memory
    if (CUT && p.push_bytes > 0) {
        // (said here, waited for by those that send, when they do)
        if (threadIdx.x == 0) expect_tx(told, groups_of(unit_of(p, first_unit, p.n_tiles).rows, cut, p.splits) * p.splits * (BM * 16));
        __syncwarp();
        cluster_arrive();
    }
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const unsigned tmem = tmem_slot;
    volatile int* aborted = &abort_flag;
    bool met = false;                  // SPLIT: whether the cluster has been waited for
    grid_launch_dependents();
    // the row of W's scales that a lane copies as number j of four, of a slab; N and beyond: none
    auto scale_row = [&](int slab, int j) {
        if (EPI != GATED) return slab * BM + 32 * j + lane;
        const int f = (slab * 4 + j) * 16 + (lane & 15);        // (lanes 0 to 15 gates, 16 to 31 their ups)
        return f < p.hidden ? f + (lane >= 16 ? p.hidden : 0) : p.N;
    };
    // Nothing is read before the kernel ahead of this one has ended: rows in 8 bits are made by kernels of this library, which let their
    // successors start early, and W is such rows.  But what a product without a list of tiles reads first is known: it comes into L2 meanwhile
    // (decode steps of 8, by 32 layers: 2.668 ms so, 2.644 when W was loaded outright, which read rows that were not there yet).
    if (p.tiles == nullptr && first_unit < p.n_tiles * p.slabs) {
        const int slab = first_unit / p.n_tiles * SIDES + rank;
        if (warp == 0 && elect_one()) {
            const int until = min(kb1, kb0 + p.stages * BOXES);
            for (int kb = kb0; kb < until; ++kb) {
                if (EPI == GATED) prefetch_box_gated(&map_w, kb * BK, slab * 4);
                else prefetch_box(&map_w, kb * BK, slab * BM);
            }
        }
        const int kb = kb0 + (warp - 2) * TURN;
        if ((warp == 2 || warp == 3) && kb < kb1) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int r = scale_row(slab, j);
                if (r < p.N) prefetch_line(p.w_scales + (long long)r * p.pitch + kb);
            }
        }
        __syncwarp();
    }
    grid_dependency_wait();

    // a slab's box: 128 rows of W, or 64 gates and their ups
    // Experts: W is read by few tiles, side by side, x by every slab: W is the first to leave L2 (2,048 tokens through gates and ups of
    // 32 experts: 1.28 GB from memory without the mark, 1.11 with it, 585,000 cycles and 524,000).
    const unsigned long long x_policy = policy_normal(), w_policy = p.tiles != nullptr ? policy_first() : x_policy;
    auto load_w = [&](unsigned at, unsigned bar, int k, int slab, int expert) {
        if (EPI == GATED) tma_load_gated<PAIR>(at, &map_w, bar, k, slab * 4, expert, w_policy);
        else tma_load<PAIR>(at, &map_w, bar, k, expert * p.N + slab * BM, w_policy);
    };
    const int n_tiles = p.tiles != nullptr ? p.tiles[0] : p.n_tiles;
    const int units = n_tiles * p.slabs;

    if (warp == 0) {
        if (elect_one()) {
            int stage = 0, issued = 0;
            unsigned phase = 1;                // (a barrier that has completed nothing counts as having completed phase 1)
            bool ok = true;
            for (int u = first_unit; u < units && ok; u += step) {
                const Unit t = unit_of(p, u, n_tiles);
                const int slab = t.slab * SIDES + rank, x_row = t.row0 + rank * (((t.rows + 15) & ~15) / 2);
                for (int kb = kb0; kb < kb1; kb += BOXES) {
                    if (!wait_one(empty + 8 * stage, phase, aborted)) {
                        give_up(aborted, p.status, ERR_TMA_WAIT);
                        ok = false;
                        break;
                    }
                    const unsigned at = smem0 + stage * stage_bytes, bar = leader(full + 8 * stage);
                    const int boxes = min(BOXES, kb1 - kb);
                    if (rank == 0) expect_tx(full + 8 * stage, SIDES * boxes * (w_bytes + p.x_box * BK));
#pragma unroll
                    for (int i = 0; i < BOXES; ++i) {
                        if (i < boxes) {
                            load_w(at + i * w_bytes, bar, (kb + i) * BK, slab, t.expert);
                            tma_load<PAIR>(at + BOXES * w_bytes + i * x_bytes, &map_x, bar, (kb + i) * BK, x_row, x_policy);
                        }
                    }
                    if (issued < p.stages) ++issued;
                    if (++stage == p.stages) { stage = 0; phase ^= 1; }
                }
            }
            // whatever happened to the others, the copies under way land before the CTA ends (a pair ends together, and the first
            // CTA's barriers count for both)
            int none = 0;
            for (int i = 0; i < issued && rank == 0; ++i) {
                if (--stage < 0) { stage = p.stages - 1; phase ^= 1; }
                wait_one(full + 8 * stage, phase ^ 1, &none);
            }
        }
        __syncwarp();
    } else if (warp == 1 && rank == 0) {
        if (elect_one()) {
            const unsigned short both = 3;         // (CTAs of the pair)
            int stage = 0, buf = 0, n = 0;
            unsigned phase = 0, sc_phase = 0, word = 0;
            bool ok = true;
            for (int u = first_unit; u < units && ok; u += step, ++n) {
                const Unit t = unit_of(p, u, n_tiles);
                const int acc = n & 1, N = (t.rows + 15) & ~15;
                const unsigned d = tmem + acc * ACC_COLS;
                if (!wait_one(acc_empty + 8 * acc, ((n >> 1) & 1) ^ 1, aborted)) {
                    give_up(aborted, p.status, ERR_MMA_WAIT);
                    break;
                }
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                for (int kb = kb0; kb < kb1; kb += BOXES) {
                    if ((kb - kb0) % TURN == 0 && !wait_one(sc_full + 8 * buf, sc_phase, aborted)) {
                        give_up(aborted, p.status, ERR_MMA_WAIT);
                        ok = false;
                        break;
                    }
                    if (kb % 4 == 0) {
                        // (two sets in turn: copies and products are carried out in the order of their issue)
                        word ^= 1;
                        const unsigned at = scales_at + buf * turn_bytes + (kb - kb0) / 4 % 4 * word_bytes, to = tmem + p.scale_col + word * p.set_cols;
                        copy_scales<PAIR>(to, scale_desc(at));
                        copy_scales<PAIR>(to + 4, scale_desc(at + 512));
                        if (N > 128) copy_scales<PAIR>(to + 8, scale_desc(at + 1024));
                    }
                    const unsigned set = tmem + p.scale_col + word * p.set_cols;
                    if (!wait_one(full + 8 * stage, phase, aborted)) {
                        give_up(aborted, p.status, ERR_MMA_WAIT);
                        ok = false;
                        break;
                    }
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    const unsigned at = smem0 + stage * stage_bytes;
#pragma unroll
                    for (int i = 0; i < BOXES; ++i) {
                        if (kb + i < kb1) {
                            const unsigned idesc = instruction(SIDES * BM, N, (kb + i) & 3);
                            const unsigned long long a = operand_desc(at + i * w_bytes), b = operand_desc(at + BOXES * w_bytes + i * x_bytes);
#pragma unroll
                            for (int k = 0; k < 4; ++k) mma<PAIR>(d, a + 2 * k, b + 2 * k, idesc, set, set + 4, (kb > kb0 || i > 0 || k > 0) ? 1u : 0u);
                        }
                    }
                    commit<PAIR>(empty + 8 * stage, both);
                    if (++stage == p.stages) { stage = 0; phase ^= 1; }
                    if ((kb - kb0) % TURN == TURN - BOXES || kb + BOXES >= kb1) {
                        commit<PAIR>(sc_empty + 8 * buf, both);
                        if (++buf == p.scale_bufs) { buf = 0; sc_phase ^= 1; }
                    }
                }
                if (ok) commit<PAIR>(acc_full + 8 * acc, both);
            }
            // (the products read shared memory and their commits write barriers: all of it ends before the CTA does)
            int none = 0;
            commit<PAIR>(drained, both);
            wait_one(drained, 0, &none);
        }
        __syncwarp();
    } else if (warp == 2 || warp == 3) {
        int turn = 0, buf = 0;
        unsigned phase = 1;
        bool ok = true;
        for (int u = first_unit; u < units && ok; u += step) {
            const Unit t = unit_of(p, u, n_tiles);
            const long long first = (long long)t.expert * p.N;
            for (int kb = kb0; kb < kb1; kb += TURN, ++turn) {
                if ((turn & 1) == warp - 2) {
                    if (!mbar_wait(sc_empty + 8 * buf, phase, aborted)) {
                        if (lane == 0) give_up(aborted, p.status, ERR_SCALE_WAIT);
                        ok = false;
                        break;
                    }
                    const unsigned at = scales_at + buf * turn_bytes + 16 * lane;
                    const int words = min(4, (kb1 - kb + 3) / 4);
                    const bool whole = kb % TURN == 0;
                    unsigned v[12][4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const int r = scale_row(t.slab * SIDES + rank, j);
                        load_words(r < p.N ? p.w_scales + (first + r) * p.pitch + kb : nullptr, words, whole && p.w_whole, v[j]);
                    }
#pragma unroll
                    for (int j = 4; j < 12; ++j) {
                        const int r = 32 * (j - 4) + lane;
                        load_words(r < t.rows ? p.x_scales + (long long)(t.row0 + r) * p.pitch + kb : nullptr, words, whole && p.x_whole, v[j]);
                    }
#pragma unroll
                    for (int j = 0; j < 12; ++j) {
                        if (j >= 4 && 32 * (j - 4) >= t.rows) break;
                        const unsigned to = at + (j < 4 ? 4 * j : 512 + (j - 4) / 4 * 512 + 4 * (j % 4));
#pragma unroll
                        for (int w = 0; w < 4; ++w)
                            if (w < words) asm volatile("st.shared.b32 [%0], %1;" ::"r"(to + w * word_bytes), "r"(v[j][w]) : "memory");
                    }
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    __syncwarp();
                    arrive_elect<PAIR>(leader(sc_full + 8 * buf));
                }
                if (++buf == p.scale_bufs) { buf = 0; phase ^= 1; }
            }
        }
    } else if (warp >= 4 && EPI == PLAIN) {
        const int quarter = warp & 3;
        constexpr int SHARES = result_warps(FORM) / 4;
        const int share = (warp - 4) >> 2;
        unsigned char* const mine = staging + (warp - 4) * 2048;
        const bool wide = !p.out_is_f32 && p.N % 8 == 0;
        int n = 0;
        for (int u = first_unit; u < units; u += step, ++n) {
            const Unit t = unit_of(p, u, n_tiles);
            const int acc = n & 1;
            if (!mbar_wait(acc_full + 8 * acc, (n / 2) & 1, aborted)) {
                if (lane == 0) give_up(aborted, p.status, ERR_EPI_WAIT);
                break;
            }
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const int first = (t.slab * SIDES + rank) * BM + quarter * 32;          // this warp's first row of W
            for (int c0 = 32 * share; c0 < t.rows; c0 += 32 * SHARES) {
                unsigned r[32];
                // (a load of 32 columns may reach into the scales' columns behind the accumulator: read, not used)
                tmem_load32(tmem + acc * ACC_COLS + ((unsigned)(quarter * 32) << 16) + c0, r);
                asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
                if (CUT && p.push_bytes > 0) {
                    if (!met) cluster_wait();          // (all barriers of the cluster are set up)
                    met = true;
#pragma unroll
                    for (int j = 0; j < 32; j += 4) {
                        const int g = (c0 + j) / 4;
                        if (c0 + j < t.rows)
                            store_async4(in_cta(smem_u32(pushed) + ((g / p.splits * p.splits + cut) * BM + quarter * 32 + lane) * 16, g % p.splits), r + j,
                                         in_cta(told, g % p.splits));
                    }
                } else if (CUT) {
                    // (every product of the CTA has been taken: the stages are free)
#pragma unroll
                    for (int j = 0; j < 32; ++j)
                        if (c0 + j < t.rows) reinterpret_cast<float*>(smem_at)[(c0 + j) * BM + quarter * 32 + lane] = __uint_as_float(r[j]);
                } else if (wide) {
                    __syncwarp();
#pragma unroll
                    for (int j = 0; j < 32; ++j)
                        *reinterpret_cast<__nv_bfloat16*>(mine + j * 64 + lane * 2) = __float2bfloat16_rn(__uint_as_float(r[j]));
                    __syncwarp();
                    // four lanes to a token: 64 bytes of its row
                    const int row = first + (lane & 3) * 8;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int tok = i * 8 + (lane >> 2);
                        const uint4 v = *reinterpret_cast<const uint4*>(mine + tok * 64 + (lane & 3) * 16);
                        if (c0 + tok < t.rows && row < p.N)
                            *reinterpret_cast<uint4*>(reinterpret_cast<__nv_bfloat16*>(p.out) + (size_t)(t.row0 + c0 + tok) * p.N + row) = v;
                    }
                } else if (first + lane < p.N) {
#pragma unroll
                    for (int j = 0; j < 32; ++j) {
                        if (c0 + j >= t.rows) break;
                        const size_t at = (size_t)(t.row0 + c0 + j) * p.N + first + lane;
                        if (p.out_is_f32) reinterpret_cast<float*>(p.out)[at] = __uint_as_float(r[j]);
                        else reinterpret_cast<__nv_bfloat16*>(p.out)[at] = __float2bfloat16_rn(__uint_as_float(r[j]));
                    }
                }
            }
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            arrive_elect<PAIR>(leader(acc_empty + 8 * acc));
            if (CUT && p.push_bytes > 0) {
                // this CTA's groups, added up in the order of K: a row of W a lane, four rows of x
                const int own = groups_of(t.rows, cut, p.splits), row = t.slab * BM + quarter * 32 + lane;
                if (own > 0 && !mbar_wait<true>(told, 0, aborted)) {
                    if (lane == 0) give_up(aborted, p.status, ERR_EPI_WAIT);
                    break;
                }
                for (int i = 0; i < own; ++i) {
                    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
                    for (int s = 0; s < p.splits; ++s) {
                        const float4 v = *reinterpret_cast<const float4*>(pushed + ((i * p.splits + s) * BM + quarter * 32 + lane) * 16);
                        if (s == 0) a = v;
                        else { a.x += v.x; a.y += v.y; a.z += v.z; a.w += v.w; }
                    }
                    const float q[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const int c = (i * p.splits + cut) * 4 + j;
                        if (c >= t.rows || row >= p.N) break;
                        const size_t at = (size_t)(t.row0 + c) * p.N + row;
                        if (p.out_is_f32) reinterpret_cast<float*>(p.out)[at] = q[j];
                        else reinterpret_cast<__nv_bfloat16*>(p.out)[at] = __float2bfloat16_rn(q[j]);
                    }
                }
            }
        }
    } else if (warp >= 4) {
        // The sums become 8-bit rows: the activation, the largest magnitude of every 128 for each row of x, the numbers under their
        // scales.  A lane has a row of W (GATED: a half warp has the gates of 16, the other half their ups; they exchange half
        // of their columns, and each lane then has 16 finished numbers of 32 columns), so the largest of a row of x is over lanes,
        // warps and, GATED, where a CTA has 64 of the 128, both CTAs.  Meanwhile the numbers lie in tensor memory, over the sums.
        constexpr int VALUES = EPI == GATED ? 16 : 32;          // finished numbers a lane and 32 columns
        const int quarter = warp & 3, odd = (warp - 4) >> 2, thread = threadIdx.x - 128;
        unsigned char* const mine = staging + (warp - 4) * 1024;
        const unsigned lanes_at = (unsigned)(quarter * 32) << 16;
        const int pitch = fp8_scale_pitch(p.hidden);
        int n = 0;
        for (int u = first_unit; u < units; u += step, ++n) {
            const Unit t = unit_of(p, u, n_tiles);
            const int acc = n & 1, slab = t.slab * SIDES + rank;
            const unsigned d = tmem + acc * ACC_COLS + lanes_at;
            bool ok = mbar_wait(acc_full + 8 * acc, (n / 2) & 1, aborted);
            if (!ok && lane == 0) give_up(aborted, p.status, ERR_EPI_WAIT);
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            // (GATED: the row of the hidden rows that a lane's numbers stand in, and whether there is one: the others are zeros, as W's rows are)
            const bool there = EPI == GATED || slab * BM + quarter * 32 + lane < p.N;
            for (int c0 = 32 * odd; ok && c0 < t.rows; c0 += 64) {
                unsigned r[32];
                tmem_load32(d + c0, r);
                asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
                for (int half = 0; half < VALUES / 16; ++half) {
                    float v[16];
#pragma unroll
                    for (int j = 0; j < 16; ++j) {
                        if (EPI == GATED) {
                            const unsigned other = __shfl_xor_sync(0xffffffffu, lane < 16 ? r[j + 16] : r[j], 16);
                            v[j] = fp8_gated(__uint_as_float(lane < 16 ? r[j] : other), __uint_as_float(lane < 16 ? other : r[j + 16]), ACTIVATION, p.gate);
                        } else {
                            v[j] = there ? fp8_act(__uint_as_float(r[16 * half + j]), ACTIVATION) : 0.f;
                        }
                    }
#pragma unroll
                    for (int j = 0; j < 16; ++j) {
                        const unsigned b = __float_as_uint(v[j]) & 0x7fffffffu;
                        const bool fine = b < 0x7f800000u;
                        r[16 * half + j] = fine ? b : 0u;
                        if (!fine) v[j] = __int_as_float(0x7fffffff);
                    }
                    // (behind a tile's last columns lie scales of products under way)
                    if (EPI == GATED || c0 + 16 * half < t.rows) tmem_store16(d + c0 + 16 * half, v);
                }
                if (EPI == GATED) {
                    unsigned m[16];
#pragma unroll
                    for (int j = 0; j < 16; ++j) m[j] = r[j];
                    tops[quarter * COLUMNS + c0 + lane] = largest_of_lanes<16>(m);        // (columns c0 .. c0 + 15 by the first half warp)
                } else {
                    tops[quarter * COLUMNS + c0 + lane] = largest_of_lanes<32>(r);
                }
            }
            asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
            if (!meet(ok)) break;
            unsigned top = 0u;
            if (thread < t.rows) {
#pragma unroll
                for (int q = 0; q < 4; ++q) top = max(top, tops[q * COLUMNS + thread]);
                // (a store that counts itself when it has landed: a fence would wait for all that the warp has stored)
                if (EPI == GATED) store_async(smem_u32(theirs + acc * COLUMNS + thread), top, told + 8 * acc, rank ^ 1);
            }
            if (EPI == GATED) {
                // (the other CTA's next store to this place is behind two units of this one)
                if (thread == 0) expect_tx(told + 8 * acc, 4 * t.rows);
                __syncwarp();
                ok = mbar_wait<true>(told + 8 * acc, (n / 2) & 1, aborted);
                if (!ok && lane == 0) give_up(aborted, p.status, ERR_EPI_WAIT);
            }
            if (thread < t.rows && ok) {
                if (EPI == GATED) top = max(top, theirs[acc * COLUMNS + thread]);
                const int e = fp8_exponent(top), block = EPI == GATED ? t.slab : slab;
                inverse[thread] = fp8_inverse(e);
                if ((EPI != GATED || rank == 0) && block * FP8_BLOCK < p.hidden) {
                    unsigned char* s = p.scales + (size_t)(t.row0 + thread) * pitch;
                    s[block] = (unsigned char)(e + 127);
                    if ((block + 1) * FP8_BLOCK >= p.hidden)
                        for (int k = block + 1; k < pitch; ++k) s[k] = 0;
                }
            }
            if (!meet(ok)) break;
            for (int c0 = 32 * odd; c0 < t.rows; c0 += 64) {
#pragma unroll
                for (int half = 0; half < VALUES / 16; ++half) {
                    unsigned r[16];
                    tmem_load16(d + c0 + 16 * half, r);
                    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
                    const int first = EPI == GATED ? (lane >> 4) * 16 : 16 * half;       // the column of r[0], from c0 on
                    __syncwarp();
#pragma unroll
                    for (int j = 0; j < 16; j += 4) {
                        const float4 inv = *reinterpret_cast<const float4*>(inverse + c0 + first + j);
                        const unsigned lo = fp8_pack2(__uint_as_float(r[j]) * inv.x, __uint_as_float(r[j + 1]) * inv.y);
                        const unsigned hi = fp8_pack2(__uint_as_float(r[j + 2]) * inv.z, __uint_as_float(r[j + 3]) * inv.w);
                        constexpr int ROW = EPI == GATED ? 16 : 32;
                        unsigned char* to = mine + (first + j) * ROW + (lane & (ROW - 1));
                        to[0] = (unsigned char)lo;
                        to[ROW] = (unsigned char)(lo >> 8);
                        to[2 * ROW] = (unsigned char)hi;
                        to[3 * ROW] = (unsigned char)(hi >> 8);
                    }
                }
                __syncwarp();
                // 16 bytes a lane: GATED, a column's 16; else half of a column's 32
#pragma unroll
                for (int i = 0; i < VALUES / 16; ++i) {
                    const int c = EPI == GATED ? lane : i * 16 + (lane >> 1);
                    const int f = EPI == GATED ? (slab * 4 + quarter) * 16 : slab * BM + quarter * 32 + (lane & 1) * 16;
                    const uint4 v = *reinterpret_cast<const uint4*>(mine + (EPI == GATED ? c * 16 : c * 32 + (lane & 1) * 16));
                    if (c0 + c < t.rows && f < p.hidden) *reinterpret_cast<uint4*>(p.codes + (size_t)(t.row0 + c0 + c) * p.hidden + f) = v;
                }
            }
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            arrive_elect<PAIR>(leader(acc_empty + 8 * acc));
        }
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    if (CUT && p.push_bytes > 0 && !met) cluster_wait();       // (every thread waits once; the result warps did when they sent)
    __syncthreads();
    // a CTA that gave up does not end before the others have (whatever they send it has somewhere to land)
    if (CUT && p.push_bytes > 0 && *aborted) cluster_sync();
    if (CUT && p.push_bytes == 0) {
        // every CTA adds up, in the order of K, the rows cut, cut + splits, .. of x's tile for its rows of W: 32 threads a row, four
        // rows of W a thread
        cluster_sync();
        const Unit t = unit_of(p, first_unit, n_tiles);
        const unsigned sums = smem0 + (threadIdx.x & 31) * 16;
        const int row = (t.slab * SIDES + rank) * BM + (threadIdx.x & 31) * 4;
        for (int c = cut + (threadIdx.x >> 5) * p.splits; c < t.rows && !*aborted; c += (threads_of(FORM) >> 5) * p.splits) {
            float4 v[8];
#pragma unroll
            for (int s = 0; s < 8; ++s)
                if (s < p.splits) v[s] = load_from(sums + c * (BM * 4), s);
            float4 a = v[0];
#pragma unroll
            for (int s = 1; s < 8; ++s)
                if (s < p.splits) { a.x += v[s].x; a.y += v[s].y; a.z += v[s].z; a.w += v[s].w; }
            const size_t at = (size_t)(t.row0 + c) * p.N + row;
            const float q[4] = {a.x, a.y, a.z, a.w};
            if (p.N % 4 == 0 && row < p.N) {
                if (p.out_is_f32) {
                    *reinterpret_cast<float4*>(reinterpret_cast<float*>(p.out) + at) = a;
                } else {
                    const __nv_bfloat162 lo = __floats2bfloat162_rn(a.x, a.y), hi = __floats2bfloat162_rn(a.z, a.w);
                    *reinterpret_cast<uint2*>(reinterpret_cast<__nv_bfloat16*>(p.out) + at) = make_uint2(reinterpret_cast<const unsigned&>(lo), reinterpret_cast<const unsigned&>(hi));
                }
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if (row + i >= p.N) break;
                    if (p.out_is_f32) reinterpret_cast<float*>(p.out)[at + i] = q[i];
                    else reinterpret_cast<__nv_bfloat16*>(p.out)[at + i] = __float2bfloat16_rn(q[i]);
                }
            }
        }
        cluster_sync();                // nobody reads this CTA's sums any more
    }
    if (PAIR && rank == 1 && warp == 1) {
        // the second CTA issues nothing, but commits arrive at its barriers too, the last of them perhaps later than at the
        // first CTA's: it must not end before they have
        int none = 0;
        mbar_wait(drained, 0, &none);
    }
    __syncwarp();
    if (PAIR) cluster_sync();          // nothing of one CTA is used by the other from here on
    if (warp == 1) {
        __syncwarp();
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        if (PAIR) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(p.tmem_cols) : "memory");
        else asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(p.tmem_cols) : "memory");
    }
    if (PAIR) {                        // the pair gives its tensor memory back together, and ends together
        __syncthreads();
        cluster_sync();
    }
}

// ---- host side ---------------------------------------------------------------------------------

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                  const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiledFn encode_tiled() {
    static EncodeTiledFn fn = nullptr;
    if (fn == nullptr) {
        void* ptr = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) == cudaSuccess && q == cudaDriverEntryPointSuccess)
            fn = reinterpret_cast<EncodeTiledFn>(ptr);
    }
    return fn;
}

// rows x K bytes, row-major; box = box_rows x 128 bytes, 128-byte swizzle, zeros outside
int make_map(CUtensorMap* map, const void* base, long long rows, long long K, int box_rows) {
    EncodeTiledFn fn = encode_tiled();
    if (fn == nullptr) return TL_BAD_SIZE;
    cuuint64_t dims[2] = {(cuuint64_t)K, (cuuint64_t)rows};
    cuuint64_t strides[1] = {(cuuint64_t)K};
    cuuint32_t box[2] = {(cuuint32_t)BK, (cuuint32_t)box_rows};
    cuuint32_t elem[2] = {1, 1};
    return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS ? TL_OK : TL_BAD_SIZE;
}

// [experts, 2 hidden, K] bytes, an expert's rows [gates; ups]: boxes of 16 gates and their 16 ups in turn, four times
int make_gated_map(CUtensorMap* map, const void* base, int experts, int hidden, long long K) {
    EncodeTiledFn fn = encode_tiled();
    if (fn == nullptr) return TL_BAD_SIZE;
    cuuint64_t dims[5] = {(cuuint64_t)K, 16, 2, (cuuint64_t)hidden / 16, (cuuint64_t)experts};
    cuuint64_t strides[4] = {(cuuint64_t)K, (cuuint64_t)hidden * K, 16 * (cuuint64_t)K, 2 * (cuuint64_t)hidden * K};
    cuuint32_t box[5] = {(cuuint32_t)BK, 16, 2, 4, 1};
    cuuint32_t elem[5] = {1, 1, 1, 1, 1};
    return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 5, const_cast<void*>(base), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS ? TL_OK : TL_BAD_SIZE;
}

constexpr int MAX_DEVICES = 64;
int current_device() {
    int dev = 0;
    return cudaGetDevice(&dev) == cudaSuccess && dev >= 0 && dev < MAX_DEVICES ? dev : 0;
}
// (asked once a device; two threads that ask at once write the same number)
int sm_count() {
    static int count[MAX_DEVICES];
    const int dev = current_device();
    if (count[dev] == 0) {
        int n = 0;
        count[dev] = cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) == cudaSuccess && n > 1 ? n : 148;
    }
    return count[dev];
}

// rows of x a tile: even shares of at most MAX_WIDTH
int even_width(int M, int most) {
    const int tiles = (M + most - 1) / most;
    return ((M + tiles - 1) / tiles + 15) / 16 * 16;
}

int whole_columns(int n) {
    int c = 32;
    while (c < n) c *= 2;
    return c;
}

template <int FORM, int EPI = PLAIN, int ACTIVATION = 0>
int launch(Params& p, const void* x, const void* w, int experts, int K, cudaStream_t s) {
    constexpr int SIDES = FORM == PAIRS ? 2 : 1;
    p.slabs = (p.N + SIDES * BM - 1) / (SIDES * BM);
    if ((long long)p.slabs * p.n_tiles * 8 > 0x7fffffffll) return TL_BAD_SIZE;
    const int units = p.slabs * p.n_tiles, sms = sm_count();
    const int stage_bytes = boxes_of(FORM) * (BM * BK + p.width / SIDES * BK);
    p.scale_bufs = FORM == SPLIT ? (p.split_blocks + TURN - 1) / TURN : MAX_SCALE_BUFS;
    if (p.scale_bufs > MAX_SCALE_BUFS) p.scale_bufs = MAX_SCALE_BUFS;
    if (FORM == SPLIT && p.width <= PUSH_WIDTH) {
        const int groups = p.width / 4;
        p.push_bytes = (groups + p.splits - 1) / p.splits * p.splits * BM * 16;
    }
    const int fixed = 1024 + p.push_bytes + p.scale_bufs * 4 * scale_bytes(p.width) + (FORM == SPLIT ? 0 : STAGING) + (EPI == PLAIN ? 0 : 7 * COLUMNS * 4);     // (1,024 to align)
    int room = 226 * 1024;                          // (a kilobyte is left for barriers)
    if (FORM == SPLIT) {
        // one accumulator, one unit: narrow tiles leave room for a second CTA on an SM
        const int sets = p.width <= 128 ? 8 : 12;
        p.scale_col = p.width;
        p.set_cols = sets;
        // (128 columns at most where there is room for another kernel's CTA: none that takes more than 384 fits beside 112 KB, so clusters
        // never wait in a circle for each other's columns)
        p.tmem_cols = whole_columns(p.width + 2 * sets);
        if (p.width <= SHARED_WIDTH && units * p.splits > sms) room = 112 * 1024;
    } else {
        p.scale_col = MAX_WIDTH;
        p.set_cols = ACC_COLS;
        p.tmem_cols = 2 * ACC_COLS;
    }
    p.stages = (room - fixed) / stage_bytes;
    if (p.stages > MAX_STAGES) p.stages = MAX_STAGES;
    if (p.stages < 1 || (FORM == SPLIT && p.push_bytes == 0 && p.stages * stage_bytes < p.width * BM * 4)) return TL_TOO_LARGE;
    // One tile: as many rows a box as there are.  (A box that reaches beyond the last row, its first eight not all there, is copied slowly: 1 to 7
    // rows of 28,672 x 4,096 25 to 26 us with boxes of 16 rows, 21 so, and 21.5 with 8 to 16 rows.)  The tile's other rows are then whatever a stage
    // holds: they make columns of the sums that nobody reads, as the rows behind an expert's last do.
    p.x_box = p.tiles == nullptr && p.n_tiles == 1 && p.M < p.width / SIDES ? p.M : p.width / SIDES;
    CUtensorMap mw, mx;
    int rc = EPI == GATED ? make_gated_map(&mw, w, experts, p.hidden, K) : make_map(&mw, w, (long long)experts * p.N, K, BM);
    if (rc != TL_OK) return rc;
    rc = make_map(&mx, x, p.M, K, p.x_box);
    if (rc != TL_OK) return rc;
    const size_t smem = fixed + (size_t)p.stages * stage_bytes;
    auto kern = gemm_fp8_kernel<FORM, EPI, ACTIVATION>;
    static bool raised[MAX_DEVICES];
    const int dev = current_device();
    if (!raised[dev]) {
        const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, 226 * 1024);
        if (e != cudaSuccess) return (int)e;
        raised[dev] = true;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(FORM == SPLIT ? SIDES * units * p.splits : SIDES * (units < sms / SIDES ? units : sms / SIDES));
    cfg.blockDim = dim3(threads_of(FORM));
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = pdl_enabled() ? 1 : 0;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = SIDES * (FORM == SPLIT ? p.splits : 1);
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = FORM == SINGLE ? 1 : 2;
    return (int)cudaLaunchKernelEx(&cfg, kern, mw, mx, p);
}

// Clusters of so many CTAs that find room at the same time, with this much shared memory a CTA: asked once.
int clusters_at_once(int ctas, int room) {
    static int known[MAX_DEVICES][2][9];
    int& n = known[current_device()][room < 200 * 1024 ? 1 : 0][ctas];
    if (n == 0) {
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(ctas * 64);
        cfg.blockDim = dim3(threads_of(SPLIT));
        cfg.dynamicSmemBytes = room;
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = ctas;
        attr[0].val.clusterDim.y = 1;
        attr[0].val.clusterDim.z = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        auto kern = gemm_fp8_kernel<SPLIT, PLAIN, 0>;
        int found = 0;
        if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, 226 * 1024) != cudaSuccess ||
            cudaOccupancyMaxActiveClusters(&found, kern, &cfg) != cudaSuccess) {
            cudaGetLastError();
            found = 128 / ctas;
        }
        n = found < 1 ? 1 : found;
    }
    return n;
}

// splits of K for `units` units: as many as let all clusters run at once (two CTAs an SM where tiles are narrow), at most eight, each
// with at least four blocks
int splits_for(int units, int k_blocks, int width) {
    const int words = (k_blocks + 3) / 4, room = (width <= SHARED_WIDTH ? 112 : 226) * 1024;
    int splits = words < 8 ? words : 8;
    while (splits > 1 && units > clusters_at_once(splits, room)) --splits;
    const int per = (words + splits - 1) / splits;
    return (words + per - 1) / per;                 // no empty split
}

// what all forms need and check; tiles == null: one weight, tiles of `width` rows
int fill(Params& p, const void* x, const void* x_scales, const void* w, const void* w_scales, int M, int N, int K, int experts, const int* tiles,
         int most_tiles, int width, int* status) {
    if (N <= 0 || K <= 0 || K % 16 != 0 || experts <= 0 || most_tiles <= 0 || (long long)experts * N > 0x7fffff00ll) return TL_BAD_SIZE;
    if (!aligned16(x) || !aligned16(w) || status == nullptr || ((uintptr_t)x_scales & 3u) != 0 || ((uintptr_t)w_scales & 3u) != 0) return TL_BAD_ALIGN;
    p = Params{};
    p.status = status;
    p.w_scales = (const unsigned char*)w_scales; p.x_scales = (const unsigned char*)x_scales;
    p.w_whole = fp8_scale_pitch(K) % 16 == 0 && aligned16(w_scales);
    p.x_whole = fp8_scale_pitch(K) % 16 == 0 && aligned16(x_scales);
    p.tiles = tiles;
    p.M = M; p.N = N; p.k_blocks = (K + BK - 1) / BK; p.pitch = fp8_scale_pitch(K);
    p.width = width;
    p.n_tiles = most_tiles;
    p.splits = 1;
    p.split_blocks = p.k_blocks;
    return TL_OK;
}

// Pairs halve what a tile of x costs in copies, and that is what wide tiles wait for (2,048 rows of 28,672 x 4,096: 222 us
// alone, 186 in pairs); narrow ones stream W, which nobody shares (8 rows: 22.3 and 22.4)
int form_for(int width) { return width > 64 ? PAIRS : SINGLE; }

int sums(const void* x, const void* x_scales, const void* w, const void* w_scales, void* out, int out_is_f32, int M, int N, int K, int experts,
         const int* tiles, int most_tiles, int width, int form, int* status, cudaStream_t s) {
    Params p;
    const int rc = fill(p, x, x_scales, w, w_scales, M, N, K, experts, tiles, most_tiles, width, status);
    if (rc != TL_OK) return rc;
    if (!aligned16(out)) return TL_BAD_ALIGN;
    if (form < 0 || form > 3 || (form == SPLIT && tiles != nullptr) || (form == SPLIT && width > MAX_SPLIT_WIDTH)) return TL_BAD_SIZE;
    p.out = out;
    p.out_is_f32 = out_is_f32;
    if (form == 0) form = form_for(width);
    if (form == SPLIT) {
        p.splits = splits_for(((N + BM - 1) / BM) * most_tiles, p.k_blocks, width);
        const int words = (p.k_blocks + 3) / 4;
        p.split_blocks = 4 * ((words + p.splits - 1) / p.splits);
        return launch<SPLIT>(p, x, w, experts, K, s);
    }
    return form == PAIRS ? launch<PAIRS>(p, x, w, experts, K, s) : launch<SINGLE>(p, x, w, experts, K, s);
}

// (so that a tile's last row, worked out as its first plus its width, and a count of tiles stay within an int)
constexpr int MOST_ROWS = 0x7fffff00;

// rows of a tile of the experts' products: twice an even share, so that most experts need one tile
int tile_rows(int pairs, int experts) {
    const long long share = (2ll * pairs + experts - 1) / (experts > 0 ? experts : 1);
    const int width = (int)(share > MAX_WIDTH ? MAX_WIDTH : (share + 15) / 16 * 16);
    return width < 16 ? 16 : width;
}

}  // namespace

// out[M, N] (float32 or bfloat16) = x . w^T for 8-bit rows x [M, K] and w [N, K] with their scales.  form: 0 the one that fits, 1 a CTA
// to a unit, 2 a pair of CTAs, 3 a cluster that shares K.
extern "C" int tl_gemm_fp8(const void* x, const void* x_scales, const void* w, const void* w_scales, void* out, int out_is_f32, int M, int N, int K,
                           int form, int* status, void* stream) {
    if (M <= 0) return TL_OK;
    if (M > MOST_ROWS || N > MOST_ROWS) return TL_BAD_SIZE;
    // Few units leave SMs idle: their K is cut among the CTAs of a cluster.  (64 rows of 4,096 x 14,336: 25 us whole, 15.9 cut; 701 of
    // 2,048 x 8,192: 23.4 in pairs, 18.2 cut; 512 of 6,144 x 4,096, 144 units: 14.7 in pairs, 20.4 cut.)
    const int narrow = even_width(M, MAX_SPLIT_WIDTH), units = ((N + BM - 1) / BM) * ((M + narrow - 1) / narrow);
    if (form == 0 && 2 * units <= sm_count() && K > 4 * BK) form = SPLIT;
    const int width = form == SPLIT ? narrow : even_width(M, MAX_WIDTH), tiles = (M + width - 1) / width;
    return sums(x, x_scales, w, w_scales, out, out_is_f32, M, N, K, 1, nullptr, tiles, width, form, status, (cudaStream_t)stream);
}

// Rows of a tile of the experts' products.
extern "C" int tl_gemm_fp8_tile_rows(int pairs, int experts) { return tile_rows(pairs, experts); }

// The experts' products: x [pairs, K] sorted by expert, w [experts, N, K], out [pairs, N]; tiles as tl_fp8_plan leaves them, with
// tl_gemm_fp8_tile_rows(pairs, experts) rows at most and most_tiles of them at most.
extern "C" int tl_gemm_fp8_experts(const void* x, const void* x_scales, const void* w, const void* w_scales, void* out, int out_is_f32, int pairs,
                                   int N, int K, int experts, const int* tiles, int most_tiles, int form, int* status,
                                   void* stream) {
    if (pairs <= 0) return TL_OK;
    if (tiles == nullptr || pairs > MOST_ROWS) return TL_BAD_SIZE;
    return sums(x, x_scales, w, w_scales, out, out_is_f32, pairs, N, K, experts, tiles, most_tiles, tile_rows(pairs, experts), form, status,
                (cudaStream_t)stream);
}

// 8-bit rows codes [M, hidden], scales [M, fp8_scale_pitch(hidden)] of act(x . w^T), w [experts, hidden, K], or, gated, of
// act(x . gate^T) * (x . up^T), w [experts, 2 hidden, K] with an expert's rows [gates; ups].  hidden % 16 == 0; act as in fp8.cuh.
// tiles == null: one expert; else as tl_gemm_fp8_experts.  form: 0, 1 or 2 (gated: 0 or 2, 128 hidden numbers lie on a pair).
extern "C" int tl_gemm_fp8_act(const void* x, const void* x_scales, const void* w, const void* w_scales, void* codes, void* scales, int M, int hidden,
                               int K, int gated, int act, float limit, float alpha, float up_offset, int experts, const int* tiles,
                               int most_tiles, int form, int* status, void* stream) {
    if (M <= 0) return TL_OK;
    if (M > MOST_ROWS || hidden <= 0 || hidden % 16 != 0 || hidden > (1 << 26) || act < 0 || act > 4 || (act == FP8_CLAMPED_SWISH && !gated) ||
        form < 0 || form > 2 || (gated && form == SINGLE))
        return TL_BAD_SIZE;
    const int width = tiles == nullptr ? even_width(M, MAX_WIDTH) : tile_rows(M, experts);
    Params p;
    const int rc = fill(p, x, x_scales, w, w_scales, M, gated ? 2 * hidden : hidden, K, experts, tiles,
                        tiles == nullptr ? (M + width - 1) / width : most_tiles, width, status);
    if (rc != TL_OK) return rc;
    if (!aligned16(codes)) return TL_BAD_ALIGN;
    p.codes = (unsigned char*)codes;
    p.scales = (unsigned char*)scales;
    p.hidden = hidden;
    p.gate = Fp8Gate{limit, alpha, up_offset};
    cudaStream_t s = (cudaStream_t)stream;
    if (form == 0) form = form_for(width);
    if (gated) {
        if (act == FP8_SILU) return launch<PAIRS, GATED, FP8_SILU>(p, x, w, experts, K, s);
        if (act == FP8_GELU_TANH) return launch<PAIRS, GATED, FP8_GELU_TANH>(p, x, w, experts, K, s);
        if (act == FP8_RELU2) return launch<PAIRS, GATED, FP8_RELU2>(p, x, w, experts, K, s);
        if (act == FP8_GELU) return launch<PAIRS, GATED, FP8_GELU>(p, x, w, experts, K, s);
        return launch<PAIRS, GATED, FP8_CLAMPED_SWISH>(p, x, w, experts, K, s);
    }
#define TL_ACT(A) return form == PAIRS ? launch<PAIRS, ACT, A>(p, x, w, experts, K, s) : launch<SINGLE, ACT, A>(p, x, w, experts, K, s)
    if (act == FP8_SILU) TL_ACT(FP8_SILU);
    if (act == FP8_GELU_TANH) TL_ACT(FP8_GELU_TANH);
    if (act == FP8_RELU2) TL_ACT(FP8_RELU2);
    TL_ACT(FP8_GELU);
#undef TL_ACT
}
