// Matrix product on the 5th-generation tensor cores for operands kept as sums of bf16 planes.
//
// A value v is held as v = v0 + v1 (+ v2), each term a bf16 that rounds what the terms before it left: 8 mantissa bits and
// a sign per term, so two terms carry 2^-17 and three all 24 bits of an FP32.  With operands A (rows x K, TA planes) and
// B (cols x K, TB planes), both K-major,
//     D[r, c] = sum over (i, j), i + j < max(TA, TB), of sum_k A_i[r, k] B_j[c, k];
// the products left out are below 2^-24 (three planes) or 2^-16 (two).  Six MMAs of K = 16 at the bf16 rate take what three
// of K = 8 at the TF32 rate take, read as many operand bytes per step and carry three more bits; bf16 planes are 6 bytes
// per value where two TF32 planes are 8.
//
// Two accumulators.  The tensor core adds into tensor memory with truncation, so what a long sum loses grows with the
// number of additions into it.  Only the product of the leading planes is large: it has an accumulator of its own (`main`),
// which gets one addition per 16 of K, and all others, 2^-8 of it and less, go to a second one (`cross`).  `main` is folded
// into an FP32 running sum in registers with round-to-nearest adds every `chunk` K blocks.  A fold takes the tensor-memory
// pipe about 1100 clocks, during which the issuer runs ahead with the cross products of the next block (5/6 of its work with
// three planes), so that folds cost next to nothing however short the chunk.
//
// Two forms of one source, as in the FP32 product (sgemm_tf32x3.cu): PAIR = the two CTAs of a cluster on one 256 x 256 tile
// with tcgen05.mma.cta_group::2 (each stages its 128 rows of A and half of the tile's rows of B), else one CTA per 128 x 128
// tile.  Warp 0 issues TMA loads, warp 1 the MMAs, warp groups 1 and 2 fold and run the epilogue.
//
// The epilogue is a class with
//     struct Args;                                              // passed by value to the kernel
//     static __device__ void block(const Args&, const TileAt&, float* patch, int lane);
// called by a warp for every 32 x 32 block of D, whose values lie in the warp's own patch[32][PATCH_LD] in shared memory.
#pragma once

#include <algorithm>
#include <atomic>

#include <cuda_bf16.h>

#include "common.cuh"
#include "tcgen05.cuh"

namespace cakeb200 {
namespace plane {

using namespace ptx;

constexpr int BK = 64;             // K per pipeline stage: 64 bf16 = one 128-byte swizzle row
constexpr int UMMA_K = 16;         // K of one tcgen05.mma kind::f16
constexpr int BM = 128;            // rows of a CTA = lanes of tensor memory
constexpr int THREADS = 384;       // warp group 0: TMA warp, MMA warp, two idle; groups 1 and 2: drain warps
constexpr int DRAIN_WARPS = 8;
constexpr int PATCH_LD = 33;       // floats per row of a 32 x 32 patch: rows and columns are both free of bank conflicts
constexpr int PLANE_BYTES = 128 * BK * 2;  // one plane of one operand per stage and CTA: 128 rows in either form
constexpr int MAX_SMEM = 232448;

template <int TA, int TB, bool PAIR>
struct Cfg {
    static constexpr int BN = PAIR ? 256 : 128;          // columns of a tile
    static constexpr int TILE_M = PAIR ? 256 : 128;      // rows of a tile
    static constexpr int STAGE_BYTES = (TA + TB) * PLANE_BYTES;
    static constexpr int PATCH_BYTES = DRAIN_WARPS * 32 * PATCH_LD * 4;
    static constexpr int FIXED = 1024 /*alignment slack*/ + 256 /*barriers*/ + PATCH_BYTES;
    static constexpr int STAGES = (MAX_SMEM - FIXED) / STAGE_BYTES > 4 ? 4 : (MAX_SMEM - FIXED) / STAGE_BYTES;
    static constexpr int SMEM = STAGES * STAGE_BYTES + FIXED;
    static constexpr int TMEM_COLS = 2 * BN;             // main, cross
    static constexpr int COLS = BN / 2;                  // columns of a drain warp: two warps share a quarter of the lanes
    static constexpr int LIMIT = TA > TB ? TA : TB;      // products (i, j) with i + j < LIMIT
    static_assert(STAGES >= 2, "two stages at least");
    static_assert((2 * STAGES + 4) * 8 + 8 <= 256, "barriers fit their block");
};

// Where a 32 x 32 block of D lies.
struct TileAt {
    int batch;
    int row, col;     // of its upper left element
    bool mirror;      // of a symmetric product, off the diagonal: the transposed block is wanted too
};

struct Problem {
    int rows, cols, K;   // of one product
    int batch;
    int symmetric;       // rows == cols and D = D^T: only tiles on and below the diagonal are computed
    int tiles_m, tiles_n, tiles;  // tiles: of one product
    int chunk;           // K blocks between folds of `main`
    int* status_word;
};

// tile `id` of a symmetric product's lower triangle, row by row
__device__ __forceinline__ void triangle(int id, int& tm, int& tn) {
    tm = (int) ((sqrtf(8.f * (float) id + 1.f) - 1.f) * 0.5f);
    while ((tm + 1) * (tm + 2) / 2 <= id) tm++;
    while (tm * (tm + 1) / 2 > id) tm--;
    tn = id - tm * (tm + 1) / 2;
}

__device__ __forceinline__ void tile_at(const Problem& p, int id, int& batch, int& tm, int& tn) {
    batch = id / p.tiles;
    const int t = id - batch * p.tiles;
    if (p.symmetric) {
        triangle(t, tm, tn);
    } else {
        tile_coords(t, p.tiles_m, p.tiles_n, CAKEB200_SCHED_MKN, 8, tm, tn);
    }
}

__host__ __device__ constexpr uint32_t idesc_bf16(int m, int n) {
    return (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t) (n >> 3) << 17) | ((uint32_t) (m >> 4) << 24);
}

template <bool PAIR>
__device__ __forceinline__ void umma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    if constexpr (PAIR)
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a),
                     "l"(b), "r"(idesc), "r"(accumulate)
                     : "memory");
    else
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a),
                     "l"(b), "r"(idesc), "r"(accumulate)
                     : "memory");
}

template <bool PAIR>
__device__ __forceinline__ void load_box(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar) {
    if constexpr (PAIR)
        asm volatile("cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
                     "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar & PAIR_LEADER_MASK)
                     : "memory");
    else
        tma_load_3d(dst, map, x, y, z, bar);
}

template <int TA, int TB, bool PAIR, class Epilogue>
__global__ void __launch_bounds__(THREADS, 1)
plane_gemm_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, const __grid_constant__ Problem p,
                  const __grid_constant__ typename Epilogue::Args ep) {
    using C = Cfg<TA, TB, PAIR>;
    constexpr int STAGES = C::STAGES, BN = C::BN;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* tiles = (uint8_t*) (((uintptr_t) smem_raw + 1023) & ~(uintptr_t) 1023);  // swizzled tiles: 1024-byte aligned
    uint64_t* bars = (uint64_t*) (tiles + STAGES * C::STAGE_BYTES);
    uint32_t* tmem_slot = (uint32_t*) (bars + 2 * STAGES + 3);
    volatile int* abort_flag = (volatile int*) (tmem_slot + 1);
    float* patches = (float*) (tiles + STAGES * C::STAGE_BYTES + 256);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = PAIR ? cluster_ctarank() : 0u;  // the even CTA of a pair issues the MMAs
    const int unit = PAIR ? (int) blockIdx.x >> 1 : (int) blockIdx.x, units = PAIR ? (int) gridDim.x >> 1 : (int) gridDim.x;
    const int all_tiles = p.tiles * p.batch, kblocks = (p.K + BK - 1) / BK;
    const uint32_t bar0 = smem_u32(bars);
    auto full_bar = [&](int s) { return bar0 + 8u * s; };
    auto empty_bar = [&](int s) { return bar0 + 8u * (STAGES + s); };
    const uint32_t main_full = bar0 + 8u * (2 * STAGES), main_empty = main_full + 8u, cross_empty = main_full + 16u;

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; s++) {
            mbar_init(full_bar(s), 1);
            mbar_init(empty_bar(s), 1);
        }
        mbar_init(main_full, 1);
        mbar_init(main_empty, (PAIR ? 2 : 1) * DRAIN_WARPS);  // one arrival per drain warp (of both CTAs of a pair)
        mbar_init(cross_empty, (PAIR ? 2 : 1) * DRAIN_WARPS);
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) tmem_alloc<PAIR>(smem_u32(tmem_slot), (uint32_t) C::TMEM_COLS);
    tcgen05_fence_before();
    sync_all_t<PAIR>();
    tcgen05_fence_after();
    const uint32_t tmem_main = *tmem_slot, tmem_cross = tmem_main + (uint32_t) BN;

    // Registers follow the roles: 384 x 168 at launch = 128 x 40 + 256 x 232.
    if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 40;");
        if (warp == 0 && lane == 0) {
            // ------------------------------------------------------- TMA producer
            int stage = 0;
            uint32_t phase = 0;
            bool ok = true;
            for (int id = unit; ok && id < all_tiles; id += units) {
                int batch, tm, tn;
                tile_at(p, id, batch, tm, tn);
                const int a_row = tm * C::TILE_M + (int) rank * BM, b_row = tn * BN + (int) rank * 128;
                for (int kb = 0; kb < kblocks; kb++) {
                    ok = mbar_wait(empty_bar(stage), phase ^ 1, abort_flag, p.status_word, 500 + stage);
                    if (!ok) break;
                    const uint32_t base = smem_u32(tiles + stage * C::STAGE_BYTES);
                    if (rank == 0) mbar_expect_tx(full_bar(stage), (PAIR ? 2 : 1) * C::STAGE_BYTES);
#pragma unroll
                    for (int i = 0; i < TA; i++) load_box<PAIR>(base + i * PLANE_BYTES, &map_a, kb * BK, a_row, i * p.batch + batch, full_bar(stage));
#pragma unroll
                    for (int j = 0; j < TB; j++) load_box<PAIR>(base + (TA + j) * PLANE_BYTES, &map_b, kb * BK, b_row, j * p.batch + batch, full_bar(stage));
                    if (++stage == STAGES) { stage = 0; phase ^= 1; }
                }
            }
            if (!ok) {
                // gave up: let the loads already issued land before the CTA goes away (bounded)
                const unsigned long long t0 = global_ns();
                if (rank == 0) {
                    for (int s = 0; s < STAGES; s++) {
                        const uint32_t armed = (s < stage) ? phase : (phase ^ 1);
                        while (!mbar_try_wait(full_bar(s), armed) && (long long) (global_ns() - t0) < 20000000LL) {}
                    }
                } else {
                    while ((long long) (global_ns() - t0) < 200000LL) __nanosleep(1000);
                }
            }
        } else if (warp == 1 && lane == 0 && rank == 0) {
            // --------------------------------------------------------- MMA issuer
            constexpr uint32_t idesc = idesc_bf16(C::TILE_M, BN);
            int stage = 0;
            uint32_t phase = 0, fold_phase = 0, tile_phase = 0;
            bool ok = true;
            for (int id = unit; ok && id < all_tiles; id += units) {
                if (C::LIMIT > 1) {
                    ok = mbar_wait(cross_empty, tile_phase ^ 1, abort_flag, p.status_word, 510);
                    if (!ok) break;
                    tile_phase ^= 1;
                }
                uint32_t cross_acc = 0, main_acc = 0;
                int in_chunk = 0;
                for (int kb = 0; kb < kblocks; kb++) {
                    ok = mbar_wait(full_bar(stage), phase, abort_flag, p.status_word, 520 + stage);
                    if (!ok) break;
                    tcgen05_fence_after();
                    const uint32_t base = smem_u32(tiles + stage * C::STAGE_BYTES);
                    // advance 16 bf16 = 32 bytes inside the 128-byte swizzle row (16-byte units)
#pragma unroll
                    for (int k = 0; k < BK / UMMA_K; k++) {
                        const uint64_t adv = (uint64_t) (k * UMMA_K * 2 >> 4);
#pragma unroll
                        for (int s = C::LIMIT - 1; s > 0; s--)  // smallest products first
#pragma unroll
                            for (int i = 0; i < TA; i++) {
                                const int j = s - i;
                                if (j < 0 || j >= TB) continue;
                                umma<PAIR>(tmem_cross, make_kmajor_sw128_desc(base + i * PLANE_BYTES) + adv,
                                           make_kmajor_sw128_desc(base + (TA + j) * PLANE_BYTES) + adv, idesc, cross_acc);
                                cross_acc = 1;
                            }
                    }
                    if (in_chunk == 0) {  // `main` starts from zero: its last fold has been read out
                        ok = mbar_wait(main_empty, fold_phase ^ 1, abort_flag, p.status_word, 530);
                        if (!ok) break;
                        fold_phase ^= 1;
                        tcgen05_fence_after();
                        main_acc = 0;
                    }
#pragma unroll
                    for (int k = 0; k < BK / UMMA_K; k++) {
                        const uint64_t adv = (uint64_t) (k * UMMA_K * 2 >> 4);
                        umma<PAIR>(tmem_main, make_kmajor_sw128_desc(base) + adv, make_kmajor_sw128_desc(base + TA * PLANE_BYTES) + adv, idesc, main_acc);
                        main_acc = 1;
                    }
                    umma_commit_t<PAIR>(empty_bar(stage));
                    if (++stage == STAGES) { stage = 0; phase ^= 1; }
                    if (++in_chunk == p.chunk || kb + 1 == kblocks) {
                        umma_commit_t<PAIR>(main_full);
                        in_chunk = 0;
                    }
                }
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 232;");
        // ------------------------------------------------- folds and the epilogue
        constexpr int COLS = C::COLS;
        const int ew = warp - 4, quarter = warp & 3, half = ew >> 2;  // a warp may only touch lanes [32 * (warp % 4), +32)
        float* patch = patches + ew * 32 * PATCH_LD;
        const uint32_t lanes = (uint32_t) (quarter * 32) << 16, columns = (uint32_t) (half * COLS);
        const int folds = (kblocks + p.chunk - 1) / p.chunk;
        float sum[COLS];
        uint32_t fold_phase = 0;
        bool ok = true;
        for (int id = unit; ok && id < all_tiles; id += units) {
            for (int f = 0; f < folds; f++) {
                ok = mbar_wait_for(main_full, fold_phase, abort_flag, p.status_word, 540, WAIT_LIMIT_NS, 32);
                ok = __all_sync(0xffffffffu, ok);  // the tensor-memory loads below need the whole warp
                if (!ok) break;
                fold_phase ^= 1;
                tcgen05_fence_after();
                float v[64];
#pragma unroll
                for (int c = 0; c < COLS; c += 64) {
                    tmem_ld64(tmem_main + lanes + columns + (uint32_t) c, v);
                    tmem_ld_wait();
                    if (f == 0) {
#pragma unroll
                        for (int j = 0; j < 64; j++) sum[c + j] = v[j];
                    } else {
#pragma unroll
                        for (int j = 0; j < 64; j++) sum[c + j] += v[j];
                    }
                }
                tcgen05_fence_before();
                if (lane == 0) mbar_arrive_t<PAIR>(main_empty);
            }
            if (!ok) break;
            if (C::LIMIT > 1) {  // the commit of the last chunk covers the cross products too
                float v[64];
#pragma unroll
                for (int c = 0; c < COLS; c += 64) {
                    tmem_ld64(tmem_cross + lanes + columns + (uint32_t) c, v);
                    tmem_ld_wait();
#pragma unroll
                    for (int j = 0; j < 64; j++) sum[c + j] += v[j];
                }
                tcgen05_fence_before();
                if (lane == 0) mbar_arrive_t<PAIR>(cross_empty);
            }
            int batch, tm, tn;
            tile_at(p, id, batch, tm, tn);
            TileAt at;
            at.batch = batch;
            at.mirror = p.symmetric && tm != tn;
            at.row = tm * C::TILE_M + (int) rank * BM + quarter * 32;
            // rolled: the sums move down by 32 registers a turn, so that the code of a block exists once (unrolled four
            // times it would run straight through from a cold instruction cache)
#pragma unroll 1
            for (int c = 0; c < COLS; c += 32) {
                at.col = tn * BN + half * COLS + c;
#pragma unroll
                for (int j = 0; j < 32; j++) patch[lane * PATCH_LD + j] = sum[j];
#pragma unroll
                for (int j = 0; j + 32 < COLS; j++) sum[j] = sum[j + 32];
                __syncwarp();
                if (at.row < p.rows && at.col < p.cols) Epilogue::block(ep, at, patch, lane);
                __syncwarp();
            }
        }
    }
    tcgen05_fence_before();
    sync_all_t<PAIR>();  // in a pair: neither CTA frees tensor memory or leaves while the other may still touch it
    if (warp == 1) {
        tcgen05_fence_after();
        tmem_free<PAIR>(tmem_main, (uint32_t) C::TMEM_COLS);
    }
}

// ------------------------------------------------------------------ epilogue helpers

// A block is read in four steps of eight rows; lane l holds eight consecutive values of row 8 s + l / 4, from 8 (l % 4) on.
// `step` s; TRANSPOSED reads the block's transpose.
template <bool TRANSPOSED>
__device__ __forceinline__ void read8(const float* patch, int lane, int s, float* v) {
    const int r = 8 * s + (lane >> 2), c = 8 * (lane & 3);
#pragma unroll
    for (int e = 0; e < 8; e++) v[e] = TRANSPOSED ? patch[(c + e) * PATCH_LD + r] : patch[r * PATCH_LD + c + e];
}

// v = v0 + v1 + ... (round to nearest), two values packed: the next term of both, which leaves the remainders in their place
__device__ __forceinline__ uint32_t next_term(float& a, float& b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    const uint32_t u = *reinterpret_cast<const uint32_t*>(&h);
    a -= __uint_as_float(u << 16);
    b -= __uint_as_float(u & 0xffff0000u);
    return u;
}

// Planes of a matrix in memory: element (r, c) of term t of product `batch` at base + ((t * batches + batch) * rows + r) * ld + c,
// ld a multiple of 8.
struct Planes {
    __nv_bfloat16* base;
    int rows, cols, ld, batches;
};

// Eight consecutive values of a row, c a multiple of 8 below p.cols: they end within the padded row.
template <int T>
__device__ __forceinline__ void store8(const Planes& p, int batch, int r, int c, const float* value) {
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; e++) v[e] = value[e];
    __nv_bfloat16* at = p.base + ((long long) batch * p.rows + r) * p.ld + c;
    const long long plane = (long long) p.batches * p.rows * p.ld;
#pragma unroll
    for (int t = 0; t < T; t++) {
        uint4 o;
        o.x = next_term(v[0], v[1]); o.y = next_term(v[2], v[3]); o.z = next_term(v[4], v[5]); o.w = next_term(v[6], v[7]);
        *reinterpret_cast<uint4*>(at + t * plane) = o;
    }
}
template <int T>
__device__ __forceinline__ void load8(const Planes& p, int batch, int r, int c, float* v) {
    const __nv_bfloat16* at = p.base + ((long long) batch * p.rows + r) * p.ld + c;
    const long long plane = (long long) p.batches * p.rows * p.ld;
#pragma unroll
    for (int e = 0; e < 8; e++) v[e] = 0.f;
#pragma unroll
    for (int t = T - 1; t >= 0; t--) {
        const uint4 o = *reinterpret_cast<const uint4*>(at + t * plane);
        const uint32_t u[4] = {o.x, o.y, o.z, o.w};
#pragma unroll
        for (int e = 0; e < 4; e++) {
            v[2 * e] += __uint_as_float(u[e] << 16);
            v[2 * e + 1] += __uint_as_float(u[e] & 0xffff0000u);
        }
    }
}

// ------------------------------------------------------------------ host side

inline int padded(int cols) { return (cols + 7) / 8 * 8; }
inline size_t plane_bytes(int terms, int batches, int rows, int cols) {
    return ((size_t) terms * batches * rows * padded(cols) * 2 + 1023) / 1024 * 1024;
}
// tensor map over planes, boxes of 128 rows x 64 values (sgemm_tf32x3.cu has the driver's entry point)
int encode_planes(CUtensorMap* map, const Planes& p, int terms);

// Whether a product runs on pairs of SMs: a 128 x 128 tile on a single SM waits for shared memory (operands of 8 KB per MMA
// of 32 clocks) and takes about as long as a 256 x 256 tile on a pair, so pairs win as soon as they need fewer rounds of
// tiles; in a single round the small tiles spread over more SMs and have half the epilogue.
inline bool use_pairs(long long tiles_single, long long tiles_pair, int sm_count) {
    return (tiles_pair + sm_count / 2 - 1) / (sm_count / 2) < (tiles_single + sm_count - 1) / sm_count;
}
inline long long count_tiles(int rows, int cols, int batch, bool symmetric, int side) {
    const long long m = (rows + side - 1) / side, n = (cols + side - 1) / side;
    return batch * (symmetric ? m * (m + 1) / 2 : m * n);
}

template <int TA, int TB, bool PAIR, class Epilogue>
int launch_form(const CUtensorMap& a, const CUtensorMap& b, Problem p, const typename Epilogue::Args& ep, int sm_count, cudaStream_t s) {
    using C = Cfg<TA, TB, PAIR>;
    auto kernel = plane_gemm_kernel<TA, TB, PAIR, Epilogue>;
    static std::atomic<unsigned long long> opted{0};  // devices whose shared-memory limit has been raised for this kernel
    int dev = 0;
    CAKE_CUDA_OK(cudaGetDevice(&dev));
    if (dev < 64 && !(opted.load() >> dev & 1)) {
        CAKE_CUDA_OK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM));
        opted |= 1ull << dev;
    }
    p.tiles_m = (p.rows + C::TILE_M - 1) / C::TILE_M;
    p.tiles_n = (p.cols + C::BN - 1) / C::BN;
    const long long tiles = p.symmetric ? (long long) p.tiles_m * (p.tiles_m + 1) / 2 : (long long) p.tiles_m * p.tiles_n;
    if (tiles * p.batch > 0x7fffffffLL) {
        set_error("the product has too many tiles");
        return CAKEB200_ERR_TOO_LARGE;
    }
    p.tiles = (int) tiles;
    const int units = (int) std::min<long long>(tiles * p.batch, PAIR ? sm_count / 2 : sm_count);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned) (PAIR ? 2 * units : units));
    cfg.blockDim = dim3(THREADS);
    cfg.dynamicSmemBytes = C::SMEM;
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = PAIR ? 2 : 1;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    CAKE_CUDA_OK(cudaLaunchKernelEx(&cfg, kernel, a, b, p, ep));
    return CAKEB200_OK;
}

template <int TA, int TB, class Epilogue>
int launch(const CUtensorMap& a, const CUtensorMap& b, const Problem& p, const typename Epilogue::Args& ep, int sm_count, cudaStream_t s) {
    const int forced = option_get(OPT_PAIR);  // 1: pairs, 2: single SMs, 0: the rule
    const bool pair = forced ? forced == 1 : use_pairs(count_tiles(p.rows, p.cols, p.batch, p.symmetric, 128), count_tiles(p.rows, p.cols, p.batch, p.symmetric, 256), sm_count);
    if (pair) return launch_form<TA, TB, true, Epilogue>(a, b, p, ep, sm_count, s);
    return launch_form<TA, TB, false, Epilogue>(a, b, p, ep, sm_count, s);
}

}  // namespace plane
}  // namespace cakeb200
