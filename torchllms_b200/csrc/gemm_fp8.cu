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
// A persistent CTA per SM walks units (a slab of 128 rows of W, a tile of rows of x), tiles fastest, so that a slab of W comes from
// memory once and the rows of x, which are fewer, from L2.  Inside a CTA (256 threads):
//   warp 0    TMA: a [128 x 128] box of W and a [width x 128] box of x a stage, 128-byte swizzle
//   warp 1    tcgen05.cp of scales (a word a row: four blocks of 128) and tcgen05.mma, four of K 32 a stage
//   warp 2    scales from memory to shared memory, in the order that tcgen05.cp wants: row r of a chunk of 128 at 16 (r % 32) + 4 (r / 32)
//   warps 4-7 results: tcgen05.ld, through shared memory to rows of C; two accumulators, so that the next unit's products run meanwhile
// Every wait is bounded: on a time-out the CTA records a code, lets its copies land, frees its tensor memory and returns.
#include "fp8.cuh"
#include <cuda.h>

namespace {

constexpr int BM = 128;              // rows of W a CTA
constexpr int BK = 128;              // bytes of K a stage: a swizzle row, and a block of numbers that share a scale
constexpr int MAX_WIDTH = 240;       // rows of x a tile: two accumulators and two sets of scales fill 512 columns
constexpr int MAX_STAGES = 12;
constexpr int SCALE_BUFS = 4;        // words of scales (512 of K) under way
constexpr int SCALE_BYTES = 512 + 1024;
constexpr int SCALE_LAG = 2;
constexpr int NTHREADS = 256;
constexpr int STAGING = 4 * 2048;    // 32 x 32 results a warp
constexpr unsigned TMEM_COLS = 512;
constexpr unsigned SCALE_COL = 240;  // scales of set s at columns 256 s + 240: 4 of W, 8 of x
constexpr unsigned long long WAIT_LIMIT_NS = 2000ull * 1000ull * 1000ull;   // two seconds, then give up

enum : int { ERR_TMA_WAIT = 601, ERR_MMA_WAIT = 602, ERR_SCALE_WAIT = 603, ERR_EPI_WAIT = 604 };

__device__ __forceinline__ unsigned smem_u32(const void* p) { return (unsigned)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void mbar_init(unsigned bar, unsigned count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count));
}
__device__ __forceinline__ bool mbar_try_wait(unsigned bar, unsigned parity) {
    unsigned ok;
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                 : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
    return ok != 0;
}
__device__ __forceinline__ unsigned long long global_ns() {
    unsigned long long t;
    asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t));
    return t;
}
// false once the limit has passed, or as soon as another role has given up; a whole warp waits together
__device__ __forceinline__ bool mbar_wait(unsigned bar, unsigned parity, volatile int* aborted) {
    bool ok = mbar_try_wait(bar, parity);
    if (!ok) {
        const unsigned long long t0 = global_ns();
        for (unsigned i = 1; !ok; ++i) {
            ok = mbar_try_wait(bar, parity);
            if (!ok && (i & 255u) == 0u && (*aborted || global_ns() - t0 > WAIT_LIMIT_NS)) break;
        }
    }
    return __all_sync(0xffffffffu, ok);
}
__device__ __forceinline__ void give_up(volatile int* aborted, int* status, int code) {
    if ((threadIdx.x & 31) == 0) {
        *aborted = 1;
        atomicExch(status, code);
    }
}
// one elected lane of a warp in step arrives
__device__ __forceinline__ void arrive_elect(unsigned bar) {
    asm volatile("{\n\t.reg .pred e;\n\telect.sync _|e, 0xffffffff;\n\t@e mbarrier.arrive.shared::cta.b64 _, [%0];\n\t}" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void expect_tx_elect(unsigned bar, unsigned bytes) {
    asm volatile("{\n\t.reg .pred e;\n\telect.sync _|e, 0xffffffff;\n\t"
                 "@e mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;\n\t}" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ void tma_load(unsigned dst, const CUtensorMap* map, unsigned bar, int x, int y) {
    asm volatile("{\n\t.reg .pred e;\n\telect.sync _|e, 0xffffffff;\n\t"
                 "@e cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];\n\t}"
                 ::"r"(dst), "l"(map), "r"(bar), "r"(x), "r"(y) : "memory");
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
__device__ __forceinline__ void mma(unsigned d, unsigned long long a, unsigned long long b, unsigned idesc, unsigned sa, unsigned sb, unsigned accumulate) {
    asm volatile("{\n\t.reg .pred p, e;\n\telect.sync _|e, 0xffffffff;\n\tsetp.ne.b32 p, %6, 0;\n\t"
                 "@e tcgen05.mma.cta_group::1.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
                 ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(sa), "r"(sb), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void copy_scales(unsigned taddr, unsigned long long desc) {
    asm volatile("{\n\t.reg .pred e;\n\telect.sync _|e, 0xffffffff;\n\t@e tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;\n\t}"
                 ::"r"(taddr), "l"(desc) : "memory");
}
__device__ __forceinline__ void commit(unsigned bar) {
    asm volatile("{\n\t.reg .pred e;\n\telect.sync _|e, 0xffffffff;\n\t"
                 "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(bar) : "memory");
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
// four bytes from memory, zeros where there is no row
__device__ __forceinline__ void copy_word(unsigned dst, const unsigned char* src, bool there) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(there ? 4 : 0) : "memory");
}

struct Params {
    void* out;                       // [M, N] (experts: rows in sorted order)
    int* status;
    const unsigned char* w_scales;   // [experts * N][pitch]
    const unsigned char* x_scales;   // [M][pitch]
    const int* tiles;                // experts: count, then (expert, first row, rows) of every tile; null: one weight, tiles of `width` rows
    int M, N, k_blocks, pitch;
    int width;                       // rows of x a tile, a multiple of 16
    int slabs, n_tiles, stages;
    int out_is_f32;
};

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

__global__ void __launch_bounds__(NTHREADS, 1) gemm_fp8_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x,
                                                               const Params p) {
    extern __shared__ unsigned char smem_raw[];
    const unsigned smem0 = (smem_u32(smem_raw) + 1023u) & ~1023u;            // tiles want 1,024-byte alignment for the swizzle
    unsigned char* const smem_at = smem_raw + (smem0 - smem_u32(smem_raw));
    const unsigned w_bytes = BM * BK, stage_bytes = w_bytes + p.width * BK;
    const unsigned scales_at = smem0 + p.stages * stage_bytes;
    unsigned char* const staging = smem_at + p.stages * stage_bytes + SCALE_BUFS * SCALE_BYTES;
    __shared__ __align__(8) unsigned long long bars[2 * MAX_STAGES + 2 * SCALE_BUFS + 5];
    __shared__ unsigned tmem_slot;
    __shared__ int abort_flag;
    const unsigned bar0 = smem_u32(bars);
    const unsigned full = bar0, empty = bar0 + 8 * MAX_STAGES, sc_full = bar0 + 16 * MAX_STAGES, sc_empty = sc_full + 8 * SCALE_BUFS;
    const unsigned acc_full = sc_empty + 8 * SCALE_BUFS, acc_empty = acc_full + 16, drained = acc_empty + 16;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        abort_flag = 0;
        for (int s = 0; s < MAX_STAGES; ++s) { mbar_init(full + 8 * s, 1); mbar_init(empty + 8 * s, 1); }
        for (int s = 0; s < SCALE_BUFS; ++s) { mbar_init(sc_full + 8 * s, 1); mbar_init(sc_empty + 8 * s, 1); }
        for (int s = 0; s < 2; ++s) { mbar_init(acc_full + 8 * s, 1); mbar_init(acc_empty + 8 * s, 4); }
        mbar_init(drained, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)), "r"(TMEM_COLS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const unsigned tmem = tmem_slot;
    volatile int* aborted = &abort_flag;
    grid_launch_dependents();
    grid_dependency_wait();

    const int n_tiles = p.tiles != nullptr ? p.tiles[0] : p.n_tiles;
    const int units = n_tiles * p.slabs;

    if (warp == 0) {
        int it = 0, stage = 0;
        bool ok = true;
        for (int u = blockIdx.x; u < units && ok; u += gridDim.x) {
            const Unit t = unit_of(p, u, n_tiles);
            for (int kb = 0; kb < p.k_blocks; ++kb, ++it) {
                if (it >= p.stages && !mbar_wait(empty + 8 * stage, (it / p.stages - 1) & 1, aborted)) {
                    give_up(aborted, p.status, ERR_TMA_WAIT);
                    ok = false;
                    break;
                }
                const unsigned at = smem0 + stage * stage_bytes;
                expect_tx_elect(full + 8 * stage, stage_bytes);
                tma_load(at, &map_w, full + 8 * stage, kb * BK, t.expert * p.N + t.slab * BM);
                tma_load(at + w_bytes, &map_x, full + 8 * stage, kb * BK, t.row0);
                if (++stage == p.stages) stage = 0;
            }
        }
        // whatever happened to the others, the copies under way land before the CTA ends
        int none = 0;
        for (int i = it > p.stages ? it - p.stages : 0; i < it; ++i) mbar_wait(full + 8 * (i % p.stages), (i / p.stages) & 1, &none);
    } else if (warp == 1) {
        int it = 0, stage = 0, group = 0, n = 0;
        bool ok = true;
        for (int u = blockIdx.x; u < units && ok; u += gridDim.x, ++n) {
            const Unit t = unit_of(p, u, n_tiles);
            const int acc = n & 1, N = (t.rows + 15) & ~15;
            const unsigned d = tmem + acc * 256;
            if (n >= 2 && !mbar_wait(acc_empty + 8 * acc, (n / 2 - 1) & 1, aborted)) {
                give_up(aborted, p.status, ERR_MMA_WAIT);
                break;
            }
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            for (int kb = 0; kb < p.k_blocks; ++kb, ++it) {
                const int buf = group % SCALE_BUFS;
                const unsigned set = tmem + (group & 1) * 256 + SCALE_COL;
                if ((kb & 3) == 0) {
                    if (!mbar_wait(sc_full + 8 * buf, (group / SCALE_BUFS) & 1, aborted)) {
                        give_up(aborted, p.status, ERR_MMA_WAIT);
                        ok = false;
                        break;
                    }
                    const unsigned at = scales_at + buf * SCALE_BYTES;
                    copy_scales(set, scale_desc(at));
                    copy_scales(set + 4, scale_desc(at + 512));
                    if (N > 128) copy_scales(set + 8, scale_desc(at + 1024));
                }
                if (!mbar_wait(full + 8 * stage, (it / p.stages) & 1, aborted)) {
                    give_up(aborted, p.status, ERR_MMA_WAIT);
                    ok = false;
                    break;
                }
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const unsigned at = smem0 + stage * stage_bytes;
                const unsigned idesc = instruction(BM, N, kb & 3);
                const unsigned long long a = operand_desc(at), b = operand_desc(at + w_bytes);
#pragma unroll
                for (int k = 0; k < 4; ++k) mma(d, a + 2 * k, b + 2 * k, idesc, set, set + 4, (kb > 0 || k > 0) ? 1u : 0u);
                commit(empty + 8 * stage);
                if (++stage == p.stages) stage = 0;
                if ((kb & 3) == 3 || kb == p.k_blocks - 1) {
                    commit(sc_empty + 8 * buf);
                    ++group;
                }
            }
            if (ok) commit(acc_full + 8 * acc);
        }
        // (the products read shared memory: they end before the CTA does)
        int none = 0;
        commit(drained);
        mbar_wait(drained, 0, &none);
    } else if (warp == 2) {
        int group = 0;
        bool ok = true;
        auto publish = [&](int g) {
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            arrive_elect(sc_full + 8 * (g % SCALE_BUFS));
        };
        for (int u = blockIdx.x; u < units && ok; u += gridDim.x) {
            const Unit t = unit_of(p, u, n_tiles);
            const long long first = (long long)t.expert * p.N;
            for (int g = 0; g * 4 < p.k_blocks; ++g, ++group) {
                const int buf = group % SCALE_BUFS;
                if (group >= SCALE_BUFS && !mbar_wait(sc_empty + 8 * buf, (group / SCALE_BUFS - 1) & 1, aborted)) {
                    give_up(aborted, p.status, ERR_SCALE_WAIT);
                    ok = false;
                    break;
                }
                const unsigned at = scales_at + buf * SCALE_BYTES + 16 * lane;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int r = t.slab * BM + 32 * j + lane;
                    const bool there = r < p.N;
                    copy_word(at + 4 * j, p.w_scales + (first + (there ? r : 0)) * p.pitch + 4 * g, there);
                }
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    if (32 * j >= t.rows) break;
                    const bool there = 32 * j + lane < t.rows;
                    copy_word(at + 512 + (j / 4) * 512 + 4 * (j % 4), p.x_scales + (long long)(t.row0 + (there ? 32 * j + lane : 0)) * p.pitch + 4 * g, there);
                }
                asm volatile("cp.async.commit_group;" ::: "memory");
                if (group >= SCALE_LAG) {
                    asm volatile("cp.async.wait_group %0;" ::"n"(SCALE_LAG) : "memory");
                    publish(group - SCALE_LAG);
                }
            }
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
        for (int g = group > SCALE_LAG ? group - SCALE_LAG : 0; g < group; ++g) publish(g);
    } else if (warp >= 4) {
        const int quarter = warp & 3;
        unsigned char* const mine = staging + quarter * 2048;
        const bool wide = !p.out_is_f32 && p.N % 8 == 0;
        int n = 0;
        for (int u = blockIdx.x; u < units; u += gridDim.x, ++n) {
            const Unit t = unit_of(p, u, n_tiles);
            const int acc = n & 1;
            if (!mbar_wait(acc_full + 8 * acc, (n / 2) & 1, aborted)) {
                give_up(aborted, p.status, ERR_EPI_WAIT);
                break;
            }
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const int first = t.slab * BM + quarter * 32;          // this warp's first row of W
            for (int c0 = 0; c0 < t.rows; c0 += 32) {
                unsigned r[32];
                // (a load of 32 columns may reach into the scales' columns behind the accumulator: read, not used)
                tmem_load32(tmem + acc * 256 + ((unsigned)(quarter * 32) << 16) + c0, r);
                asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
                if (wide) {
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
            arrive_elect(acc_empty + 8 * acc);
        }
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (warp == 1) {
        __syncwarp();
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(TMEM_COLS) : "memory");
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

int sm_count() {
    int dev = 0, n = 148;
    if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
    return n;
}

// rows of x a tile: even shares of at most MAX_WIDTH
int even_width(int M) {
    const int tiles = (M + MAX_WIDTH - 1) / MAX_WIDTH;
    return ((M + tiles - 1) / tiles + 15) / 16 * 16;
}

int launch(const void* x, const void* x_scales, const void* w, const void* w_scales, void* out, int out_is_f32, int M, int N, int K, int experts,
           const int* tiles, int most_tiles, int width, int* status, cudaStream_t s) {
    if (N <= 0 || K <= 0 || K % 16 != 0 || experts <= 0 || (long long)experts * N > 0x7fffff00ll) return TL_BAD_SIZE;
    if (!aligned16(x) || !aligned16(w) || !aligned16(out) || status == nullptr || ((uintptr_t)x_scales & 3u) != 0 || ((uintptr_t)w_scales & 3u) != 0)
        return TL_BAD_ALIGN;
    Params p = {};
    p.out = out; p.status = status; p.out_is_f32 = out_is_f32;
    p.w_scales = (const unsigned char*)w_scales; p.x_scales = (const unsigned char*)x_scales;
    p.tiles = tiles;
    p.M = M; p.N = N; p.k_blocks = (K + BK - 1) / BK; p.pitch = fp8_scale_pitch(K);
    p.width = width;
    p.slabs = (N + BM - 1) / BM;
    p.n_tiles = most_tiles;
    if ((long long)p.slabs * most_tiles > 0x7fffffffll) return TL_BAD_SIZE;
    const int most = 227 * 1024 - 1024 - 1024 - SCALE_BUFS * SCALE_BYTES - STAGING;       // (a kilobyte for barriers, one to align)
    p.stages = most / (BM * BK + width * BK);
    if (p.stages > MAX_STAGES) p.stages = MAX_STAGES;
    CUtensorMap mw, mx;
    int rc = make_map(&mw, w, (long long)experts * N, K, BM);
    if (rc != TL_OK) return rc;
    rc = make_map(&mx, x, M, K, width);
    if (rc != TL_OK) return rc;
    const size_t smem = 1024 + (size_t)p.stages * (BM * BK + width * BK) + SCALE_BUFS * SCALE_BYTES + STAGING;
    cudaError_t e = cudaFuncSetAttribute(gemm_fp8_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 226 * 1024);
    if (e != cudaSuccess) return (int)e;
    const int units = p.slabs * most_tiles, sms = sm_count();
    return (int)tl_launch(gemm_fp8_kernel, dim3(units < sms ? units : sms), dim3(NTHREADS), smem, s, mw, mx, p);
}

}  // namespace

// out[M, N] (float32 or bfloat16) = x . w^T for 8-bit rows x [M, K] and w [N, K] with their scales.
extern "C" int tl_gemm_fp8(const void* x, const void* x_scales, const void* w, const void* w_scales, void* out, int out_is_f32, int M, int N, int K,
                           int* status, void* stream) {
    if (M <= 0) return TL_OK;
    const int width = even_width(M);
    return launch(x, x_scales, w, w_scales, out, out_is_f32, M, N, K, 1, nullptr, (M + width - 1) / width, width, status, (cudaStream_t)stream);
}

// Rows of a tile of the experts' products, and how many tiles there can be.
extern "C" int tl_gemm_fp8_tile_rows(int pairs, int experts) {
    // twice an even share, so that most experts need one tile
    const long long share = (2ll * pairs + experts - 1) / (experts > 0 ? experts : 1);
    const int width = (int)(share > MAX_WIDTH ? MAX_WIDTH : (share + 15) / 16 * 16);
    return width < 16 ? 16 : width;
}

// The experts' products: x [pairs, K] sorted by expert, w [experts, N, K], out [pairs, N]; tiles as moe_plan leaves them, with
// tl_gemm_fp8_tile_rows(pairs, experts) rows at most and most_tiles of them at most.
extern "C" int tl_gemm_fp8_experts(const void* x, const void* x_scales, const void* w, const void* w_scales, void* out, int out_is_f32, int pairs,
                                   int N, int K, int experts, const int* tiles, int most_tiles, int* status, void* stream) {
    if (pairs <= 0) return TL_OK;
    if (tiles == nullptr || most_tiles <= 0) return TL_BAD_SIZE;
    return launch(x, x_scales, w, w_scales, out, out_is_f32, pairs, N, K, experts, tiles, most_tiles, tl_gemm_fp8_tile_rows(pairs, experts), status,
                  (cudaStream_t)stream);
}
