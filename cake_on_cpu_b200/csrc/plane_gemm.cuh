// Matrix product on the 5th-generation tensor cores for operands kept as sums of 16-bit planes.
//
// A value v is held as v = v0 + f v1 (+ f^2 v2), each term a 16-bit number that rounds what the terms before it left.
//   Fp16Planes: f = 2^-11, so that the second term has the range of the first; two terms carry 22 bits and a sign.  Absolute
//       resolution 2^-36, for data whose scale is known (below 2^16).
//   Bf16Planes: f = 1 and the range of FP32; two terms carry 16 bits and a sign, three all 24 bits of an FP32.
// With operands A (rows x K, TA planes) and B (cols x K, TB planes), both K-major,
//     D[r, c] = sum over (i, j), i + j < max(TA, TB), of f^(i+j) sum_k A_i[r, k] B_j[c, k];
// what is left out is of the size of the terms' own rounding.  Two FP16 terms take three MMAs at the 16-bit rate per product,
// half of what FP32 operands split into two TF32 terms take.
//
// Two accumulators.  The tensor core adds into tensor memory with truncation, so what a long sum loses grows with the
// number of additions into it.  Only the product of the leading planes is large: it has an accumulator of its own (`main`),
// which gets one addition per 16 of K, and all others go to a second one (`cross`; this is also where f is applied once).
// `main` is folded into an FP32 running sum in registers with round-to-nearest adds every `chunk` K blocks.  A fold takes
// the tensor-memory pipe about 1100 clocks, during which the issuer runs ahead with the cross products of the next block.
//
// Two forms of one source, as in the FP32 product (sgemm_tf32x3.cu): PAIR = two CTAs on one 256 x 256 tile with
// tcgen05.mma.cta_group::2 (each stages its 128 rows of A and half of the tile's rows of B), else one CTA per 128 x 128
// tile.  A 128 x 128 x 16 MMA reads 8 KB of shared memory in its 64 clocks, all an SM delivers, and TMA writes come on
// top: with two planes a K block of 64 takes 1280 clocks at best.  A pair's 256 x 256 x 16 takes 128 clocks for the same
// 8 KB per SM: 1536 clocks per K block for twice the work per SM.
//
// Few tiles.  Where a product has fewer tiles than the machine has SMs, `splits` units (CTAs or pairs) of one cluster
// share a tile: each takes a range of K, then every 32 x 32 block of the partial sums goes through distributed shared memory
// to the unit that finishes it, which adds the parts in unit order.  The epilogue is shared out with it.
//
// Warp 0 issues TMA loads, warp 1 the MMAs, warp groups 1 and 2 fold and run the epilogue, a class with
//     struct Args;                                              // passed by value to the kernel
//     static __device__ void block(const Args&, const TileAt&, const float* v, uint32_t* patch, int lane);
// called by a warp for every 32 x 32 block of D: lane l holds row l of it in v[32], and patch[32][PATCH_LD] is the warp's own
// shared memory.
//
// Kernels that follow one another may start early (programmatic launch): what a kernel sets up before it touches memory
// overlaps the end of the one before.
#pragma once

#include <algorithm>
#include <atomic>

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"
#include "tcgen05.cuh"

namespace cakeb200 {
namespace plane {

using namespace ptx;

constexpr int BK = 64;             // K per pipeline stage: 64 16-bit values = one 128-byte swizzle row
constexpr int UMMA_K = 16;         // K of one tcgen05.mma kind::f16
constexpr int BM = 128;            // rows of a CTA = lanes of tensor memory
constexpr int THREADS = 384;       // warp group 0: TMA warp, MMA warp, two idle; groups 1 and 2: drain warps
constexpr int DRAIN_WARPS = 8;
constexpr int PATCH_LD = 33;       // floats per row of a 32 x 32 patch: rows and columns are both free of bank conflicts
constexpr int PLANE_BYTES = 128 * BK * 2;  // one plane of one operand per stage and CTA: 128 rows in either form
constexpr int MAX_SMEM = 232448;
constexpr int PATCH_FLOATS = 32 * PATCH_LD;
constexpr int MAX_CLUSTER = 8;     // CTAs

struct Fp16Planes {
    static constexpr uint32_t FORMAT = 0;             // of A and B in the instruction descriptor
    static constexpr float TERM = 2048.f;             // a term counts 1 / TERM of the one before it
    // the next term of two values, packed; leaves the remainders, scaled up, in their place
    static __device__ __forceinline__ uint32_t next(float& a, float& b) {
        const __half2 h = __floats2half2_rn(a, b);
        const float2 f = __half22float2(h);
        a = (a - f.x) * TERM;
        b = (b - f.y) * TERM;
        return *reinterpret_cast<const uint32_t*>(&h);
    }
    static __device__ __forceinline__ float2 value(uint32_t u) { return __half22float2(*reinterpret_cast<const __half2*>(&u)); }
};
struct Bf16Planes {
    static constexpr uint32_t FORMAT = 1;
    static constexpr float TERM = 1.f;
    static __device__ __forceinline__ uint32_t next(float& a, float& b) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        const uint32_t u = *reinterpret_cast<const uint32_t*>(&h);
        a -= __uint_as_float(u << 16);
        b -= __uint_as_float(u & 0xffff0000u);
        return u;
    }
    static __device__ __forceinline__ float2 value(uint32_t u) { return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u)); }
};

template <int TA, int TB, bool PAIR>
struct Cfg {
    static constexpr int BN = PAIR ? 256 : 128;          // columns of a tile
    static constexpr int TILE_M = PAIR ? 256 : 128;      // rows of a tile
    static constexpr int STAGE_BYTES = (TA + TB) * PLANE_BYTES;
    static constexpr int PATCH_BYTES = DRAIN_WARPS * PATCH_FLOATS * 4;
    static constexpr int BLOCKS = 4 * BN / 32;           // 32 x 32 blocks of a CTA's part of the tile
    static constexpr int FIXED = 1024 /*alignment slack*/ + 256 /*barriers*/ + PATCH_BYTES;
    static constexpr int STAGES = (MAX_SMEM - FIXED) / STAGE_BYTES > 4 ? 4 : (MAX_SMEM - FIXED) / STAGE_BYTES;
    static constexpr int SMEM = STAGES * STAGE_BYTES + FIXED;
    static constexpr int TMEM_COLS = 2 * BN;             // main, cross
    static constexpr int COLS = BN / 2;                  // columns of a drain warp: two warps share a quarter of the lanes
    static constexpr int LIMIT = TA > TB ? TA : TB;      // products (i, j) with i + j < LIMIT
    static_assert(STAGES >= 2, "two stages at least");
    static_assert((2 * STAGES + 4) * 8 + 8 <= 256, "barriers fit their block");
    static_assert(BLOCKS * 4096 <= STAGES * STAGE_BYTES, "the parts of a shared tile fit the stages");
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
    int splits;          // units of a cluster that share a tile; > 1: one tile per cluster
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

// D = F32, A and B of one 16-bit format, both K-major
__host__ __device__ constexpr uint32_t idesc_16(uint32_t format, int m, int n) {
    return (1u << 4) | (format << 7) | (format << 10) | ((uint32_t) (n >> 3) << 17) | ((uint32_t) (m >> 4) << 24);
}

// arrives on the barrier at this offset in this CTA, or in both CTAs of this pair, once the MMAs issued so far are done
template <bool PAIR>
__device__ __forceinline__ void commit(uint32_t bar, uint32_t cluster_rank) {
    if constexpr (PAIR)
        asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar),
                     "h"((uint16_t) (3u << (cluster_rank & ~1u)))
                     : "memory");
    else
        umma_commit(bar);
}
__device__ __forceinline__ uint32_t remote_address(uint32_t local, uint32_t cluster_rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(local), "r"(cluster_rank));
    return r;
}
__device__ __forceinline__ void store_remote(uint32_t addr, const float* v) {
    asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]) : "memory");
}
// the kernel before this one in the stream has finished and its results are visible; the next one may be set up
__device__ __forceinline__ void wait_for_previous_kernel() {
    asm volatile("griddepcontrol.wait;\n\tgriddepcontrol.launch_dependents;" ::: "memory");
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

template <class Format, int TA, int TB, bool PAIR, class Epilogue>
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
    const bool clustered = PAIR || p.splits > 1;
    const uint32_t cluster_rank = clustered ? cluster_ctarank() : 0u;
    const uint32_t rank = PAIR ? cluster_rank & 1u : 0u;             // the even CTA of a pair issues the MMAs
    const int split = (int) (PAIR ? cluster_rank >> 1 : cluster_rank);  // which part of K
    // units walk the tiles in turn; the units of a shared tile are the members of one cluster
    const int per_tile = (PAIR ? 2 : 1) * p.splits;
    const int unit = (int) blockIdx.x / per_tile, units = (int) gridDim.x / per_tile;
    const int all_tiles = p.tiles * p.batch, all_blocks = (p.K + BK - 1) / BK;
    const int kb_first = (int) ((long long) all_blocks * split / p.splits), kb_end = (int) ((long long) all_blocks * (split + 1) / p.splits);
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
    if (threadIdx.x == 64) {
        asm volatile("prefetch.tensormap [%0];" ::"l"(&map_a) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&map_b) : "memory");
    }
    if (warp == 1) tmem_alloc<PAIR>(smem_u32(tmem_slot), (uint32_t) C::TMEM_COLS);
    tcgen05_fence_before();
    if (clustered) cluster_sync_all();
    else __syncthreads();
    tcgen05_fence_after();
    wait_for_previous_kernel();
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
                for (int kb = kb_first; kb < kb_end; kb++) {
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
            constexpr uint32_t idesc = idesc_16(Format::FORMAT, C::TILE_M, BN);
            int stage = 0;
            uint32_t phase = 0, fold_phase = 0, tile_phase = 0;
            bool ok = true;
            for (int id = unit; ok && id < all_tiles; id += units) {
                ok = mbar_wait(cross_empty, tile_phase ^ 1, abort_flag, p.status_word, 510);
                if (!ok) break;
                tile_phase ^= 1;
                tcgen05_fence_after();
                uint32_t cross_acc = 0, main_acc = 0;
                int in_chunk = 0;
                for (int kb = kb_first; kb < kb_end; kb++) {
                    ok = mbar_wait(full_bar(stage), phase, abort_flag, p.status_word, 520 + stage);
                    if (!ok) break;
                    tcgen05_fence_after();
                    const uint32_t base = smem_u32(tiles + stage * C::STAGE_BYTES);
                    // advance 16 values = 32 bytes inside the 128-byte swizzle row (16-byte units)
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
                    commit<PAIR>(empty_bar(stage), cluster_rank);
                    if (++stage == STAGES) { stage = 0; phase ^= 1; }
                    if (++in_chunk == p.chunk || kb + 1 == kb_end) {
                        commit<PAIR>(main_full, cluster_rank);
                        in_chunk = 0;
                    }
                }
            }
        }
        __syncwarp();
        if (p.splits > 1) {  // the two barriers of the exchange below
            cluster_sync_all();
            cluster_sync_all();
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 232;");
        // ------------------------------------------------- folds and the epilogue
        constexpr int COLS = C::COLS;
        const int ew = warp - 4, quarter = warp & 3, half = ew >> 2;  // a warp may only touch lanes [32 * (warp % 4), +32)
        float* patch = patches + ew * PATCH_FLOATS;
        const uint32_t lanes = (uint32_t) (quarter * 32) << 16, columns = (uint32_t) (half * COLS);
        const int folds = (kb_end - kb_first + p.chunk - 1) / p.chunk;
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
                const int steps = min(p.chunk, kb_end - kb_first - f * p.chunk) * (BK / UMMA_K);
                // Truncation of a sum of n additions that grow it evenly loses half a unit in the last place each time, on
                // average over the mantissas 0.36 2^-23 of the sum so far, (n + 1) / 2 times that of the last one: the part
                // of it that has a sign is put back here (measured on 4096 x 4096 FP32: error 2.0e-6 -> 1.3e-6).
                const float up = 1.f + 0.18f * 1.1920929e-7f * (float) (steps + 1);
                float v[64];
#pragma unroll
                for (int c = 0; c < COLS; c += 64) {
                    tmem_ld64(tmem_main + lanes + columns + (uint32_t) c, v);
                    tmem_ld_wait();
                    if (f == 0) {
#pragma unroll
                        for (int j = 0; j < 64; j++) sum[c + j] = v[j] * up;
                    } else {
#pragma unroll
                        for (int j = 0; j < 64; j++) sum[c + j] = fmaf(v[j], up, sum[c + j]);
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
                    for (int j = 0; j < 64; j++) sum[c + j] = fmaf(v[j], 1.f / Format::TERM, sum[c + j]);
                }
                tcgen05_fence_before();
            }
            if (lane == 0) mbar_arrive_t<PAIR>(cross_empty);
            if (p.splits > 1) break;  // one tile per cluster: on to the exchange
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
                if (at.row < p.rows && at.col < p.cols) Epilogue::block(ep, at, sum, (uint32_t*) patch, lane);
#pragma unroll
                for (int j = 0; j + 32 < COLS; j++) sum[j] = sum[j + 32];
                __syncwarp();
            }
        }
        if (p.splits > 1) {
            // Block b of a CTA's part of the tile is finished by unit b mod splits, which gets the parts of all units in its
            // stage buffers: part s of its i-th block is the (i * splits + s)-th run of 32 x 32 values.
            cluster_sync_all();  // every unit is done with its stages
            const int S = p.splits;
#pragma unroll 1
            for (int c = 0; ok && c < COLS; c += 32) {
                const int b = (half * (COLS / 32) + c / 32) * 4 + quarter;
#pragma unroll
                for (int j = 0; j < 32; j++) patch[lane * PATCH_LD + j] = sum[j];
#pragma unroll
                for (int j = 0; j + 32 < COLS; j++) sum[j] = sum[j + 32];
                __syncwarp();
                // through the patch, so that a store covers four whole rows of 128 bytes: remote shared memory is written
                // in such segments (stores of one element in each of 32 rows took 50 us per tile).  Within its row a 16-byte
                // piece is moved by the row number, so that the reader below, a row per lane, meets no bank conflicts.
                const uint32_t to = remote_address(smem_u32((float*) tiles + (b / S * S + split) * 1024), (uint32_t) (b % S) * (PAIR ? 2u : 1u) + rank);
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const int r = 4 * i + (lane >> 3), piece = lane & 7;
                    const float* from = patch + r * PATCH_LD + 4 * piece;
                    const float v[4] = {from[0], from[1], from[2], from[3]};
                    store_remote(to + 128u * r + 16u * (piece ^ (r & 7)), v);
                }
                __syncwarp();
            }
            cluster_sync_all();
            int batch, tm, tn;
            tile_at(p, unit, batch, tm, tn);
            TileAt at;
            at.batch = batch;
            at.mirror = p.symmetric && tm != tn;
#pragma unroll 1
            for (int i = ew; ok && i < C::BLOCKS / S; i += DRAIN_WARPS) {
                const int b = i * S + split;
                const float4* parts = (const float4*) ((const float*) tiles + i * S * 1024 + lane * 32);
                float v[32];
#pragma unroll
                for (int q = 0; q < 8; q++) {
                    float4 t = parts[q ^ (lane & 7)];
                    for (int s = 1; s < S; s++) {
                        const float4 u = parts[s * 256 + (q ^ (lane & 7))];
                        t.x += u.x; t.y += u.y; t.z += u.z; t.w += u.w;
                    }
                    v[4 * q] = t.x; v[4 * q + 1] = t.y; v[4 * q + 2] = t.z; v[4 * q + 3] = t.w;
                }
                at.row = tm * C::TILE_M + (int) rank * BM + (b & 3) * 32;
                at.col = tn * BN + (b >> 2) * 32;
                if (at.row < p.rows && at.col < p.cols) Epilogue::block(ep, at, v, (uint32_t*) patch, lane);
                __syncwarp();
            }
        }
    }
    tcgen05_fence_before();
    // nobody frees tensor memory or leaves while another CTA of its pair may still touch it
    if (clustered) cluster_sync_all();
    else __syncthreads();
    if (warp == 1) {
        tcgen05_fence_after();
        tmem_free<PAIR>(tmem_main, (uint32_t) C::TMEM_COLS);
    }
}

// ------------------------------------------------------------------ epilogue helpers

// Planes of a matrix in memory: element (r, c) of term t of product `batch` at base + ((t * batches + batch) * rows + r) * ld + c,
// ld a multiple of 16.
struct Planes {
    uint16_t* base;
    int rows, cols, ld, batches;
};

// Eight consecutive values of a row, c a multiple of 8 below p.cols: they end within the padded row.
template <class Format, int T>
__device__ __forceinline__ void store8(const Planes& p, int batch, int r, int c, const float* value) {
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; e++) v[e] = value[e];
    uint16_t* at = p.base + ((long long) batch * p.rows + r) * p.ld + c;
    const long long plane = (long long) p.batches * p.rows * p.ld;
#pragma unroll
    for (int t = 0; t < T; t++) {
        uint4 o;
        o.x = Format::next(v[0], v[1]); o.y = Format::next(v[2], v[3]); o.z = Format::next(v[4], v[5]); o.w = Format::next(v[6], v[7]);
        *reinterpret_cast<uint4*>(at + t * plane) = o;
    }
}
__device__ __forceinline__ void store32b(void* p, const uint32_t* v) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]),
                 "r"(v[6]), "r"(v[7])
                 : "memory");
}
__device__ __forceinline__ void load32b(const void* p, uint32_t* v) {
    asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7])
                 : "l"(p));
}

// A block's two planes and those of its transpose, 32 bytes (a whole sector) per lane and store: a lane has its row in
// registers, for the transpose the pairs of terms of a value go through the patch as one word.  direct / mirrored: where the block
// and its transpose begin, (row, col) and (mirror_row, mirror_col); padding columns get what the products of zero rows are.
template <class Format>
__device__ __forceinline__ void store_block(const float* value, float f, const Planes& p, int batch, int row, int col, const Planes& mirror, int mirror_row,
                                            int mirror_col, bool mirrored, uint32_t* patch, int lane) {
    const long long plane = (long long) p.batches * p.rows * p.ld;
    uint16_t* at = p.base + ((long long) batch * p.rows + row + lane) * p.ld + col;
#pragma unroll
    for (int h = 0; h < 2; h++) {
        uint32_t t0[8], t1[8];
#pragma unroll
        for (int i = 0; i < 8; i++) {
            float a = f * value[16 * h + 2 * i], b = f * value[16 * h + 2 * i + 1];
            t0[i] = Format::next(a, b);
            t1[i] = Format::next(a, b);
        }
        if (row + lane < p.rows && col + 16 * h < p.cols) {
            store32b(at + 16 * h, t0);
            store32b(at + 16 * h + plane, t1);
        }
        if (mirrored) {
#pragma unroll
            for (int i = 0; i < 8; i++) {
                patch[lane * PATCH_LD + 16 * h + 2 * i] = __byte_perm(t0[i], t1[i], 0x5410);
                patch[lane * PATCH_LD + 16 * h + 2 * i + 1] = __byte_perm(t0[i], t1[i], 0x7632);
            }
        }
    }
    if (!mirrored) return;
    __syncwarp();
    const long long mirror_plane = (long long) mirror.batches * mirror.rows * mirror.ld;
#pragma unroll
    for (int h = 0; h < 2; h++) {
        const int r = 16 * h + (lane >> 1), c = 16 * (lane & 1);  // 16 values of row r of the transpose
        uint32_t w[16], t0[8], t1[8];
#pragma unroll
        for (int e = 0; e < 16; e++) w[e] = patch[(c + e) * PATCH_LD + r];
#pragma unroll
        for (int i = 0; i < 8; i++) {
            t0[i] = __byte_perm(w[2 * i], w[2 * i + 1], 0x5410);
            t1[i] = __byte_perm(w[2 * i], w[2 * i + 1], 0x7632);
        }
        if (mirror_row + r < mirror.rows && mirror_col + c < mirror.cols) {
            uint16_t* to = mirror.base + ((long long) batch * mirror.rows + mirror_row + r) * mirror.ld + mirror_col + c;
            store32b(to, t0);
            store32b(to + mirror_plane, t1);
        }
    }
}

// Row `row` + lane of a block of two planes, from column `col` on; zeros outside.
template <class Format>
__device__ __forceinline__ void load_block(const Planes& p, int batch, int row, int col, int lane, float* v) {
    const long long plane = (long long) p.batches * p.rows * p.ld;
    const uint16_t* at = p.base + ((long long) batch * p.rows + row + lane) * p.ld + col;
    uint32_t t0[16], t1[16];
#pragma unroll
    for (int h = 0; h < 2; h++) {
        if (row + lane < p.rows && col + 16 * h < p.cols) {
            load32b(at + 16 * h, t0 + 8 * h);
            load32b(at + 16 * h + plane, t1 + 8 * h);
        } else {
#pragma unroll
            for (int i = 0; i < 8; i++) t0[8 * h + i] = t1[8 * h + i] = 0u;
        }
    }
#pragma unroll
    for (int i = 0; i < 16; i++) {
        const float2 a = Format::value(t0[i]), b = Format::value(t1[i]);
        v[2 * i] = fmaf(b.x, 1.f / Format::TERM, a.x);
        v[2 * i + 1] = fmaf(b.y, 1.f / Format::TERM, a.y);
    }
}

// A block through the patch to a lane per column: f(r, value) for every row r of the block, whole rows at a time.
template <typename F>
__device__ __forceinline__ void by_rows(const float* v, uint32_t* patch, int lane, F f) {
#pragma unroll
    for (int j = 0; j < 32; j++) patch[lane * PATCH_LD + j] = __float_as_uint(v[j]);
    __syncwarp();
#pragma unroll 8
    for (int r = 0; r < 32; r++) f(r, __uint_as_float(patch[r * PATCH_LD + lane]));
}

// ------------------------------------------------------------------ host side

inline int padded(int cols) { return (cols + 15) / 16 * 16; }  // rows start on whole 32-byte sectors
inline size_t plane_bytes(int terms, int batches, int rows, int cols) {
    return ((size_t) terms * batches * rows * padded(cols) * 2 + 1023) / 1024 * 1024;
}
// tensor map over planes, boxes of 128 rows x 64 values
template <class Format>
int encode_planes(CUtensorMap* map, const Planes& p, int terms) {
    const unsigned long long dims[3] = {(unsigned long long) p.cols, (unsigned long long) p.rows, (unsigned long long) terms * p.batches};
    const unsigned long long strides[2] = {(unsigned long long) p.ld * 2, (unsigned long long) p.ld * 2 * p.rows};
    const unsigned box[3] = {BK, 128, 1};
    return encode_tiled_16(map, Format::FORMAT == 1, p.base, 3, dims, strides, box, true);
}

inline long long count_tiles(int rows, int cols, int batch, bool symmetric, int side) {
    const long long m = (rows + side - 1) / side, n = (cols + side - 1) / side;
    return batch * (symmetric ? m * (m + 1) / 2 : m * n);
}

// Form of a product and the number of units that share a tile: the shortest by a model of its time in clocks.  A K block
// takes 1280 clocks on a single SM and 1536 on a pair (two planes each, see above).  What follows the last one was measured:
// 6000 clocks for the epilogue of a 128 x 128 tile, 13000 for a CTA's half of a 256 x 256 one, 12000 and 18000 with an
// exchange (its barriers, the stores, and code that a launch runs once, straight from L2).  Clusters of c CTAs fit the
// machine's GPCs about 148 / 74 / 36 / 16 times for c = 1, 2, 4, 8.
struct Form {
    bool pair;
    int splits;
};
inline Form pick_form(int rows, int cols, int K, int batch, bool symmetric, int sm_count) {
    const int forced_pair = option_get(OPT_PAIR), forced_splits = option_get(OPT_K_PIECES);  // 1: pairs, 2: single SMs; 0: this rule
    const int blocks = (K + BK - 1) / BK;
    Form best = {false, 1};
    double best_time = 1e30;
    for (int pair = 0; pair < 2; pair++) {
        if (forced_pair && (forced_pair == 1) != (pair == 1)) continue;
        const long long tiles = count_tiles(rows, cols, batch, symmetric, pair ? 256 : 128);
        const int most = std::min(blocks, MAX_CLUSTER / (pair ? 2 : 1));
        for (int splits = 1; splits <= most; splits *= 2) {
            if (forced_splits && splits * 2 <= std::min(forced_splits, most)) continue;  // forced: the largest allowed
            if (forced_splits && splits > forced_splits) break;
            const int ctas = splits * (pair ? 2 : 1);
            const int fit = ctas == 1 ? sm_count : ctas == 2 ? sm_count / 2 : ctas == 4 ? sm_count / 4 - 1 : sm_count / 8 - 2;
            const long long rounds = (tiles + fit - 1) / std::max(fit, 1);
            const double per_tile = (double) ((blocks + splits - 1) / splits) * (pair ? 1536 : 1280);
            const double epilogue = splits > 1 ? (pair ? 18000 : 12000) : (pair ? 13000 : 6000);
            // tiles of a persistent unit overlap their epilogues with the next tile's products; shared tiles do not
            const double time = splits > 1 ? rounds * (per_tile + epilogue) : rounds * (per_tile + 1500) + epilogue;
            if (time < best_time) {
                best_time = time;
                best.pair = pair != 0;
                best.splits = splits;
            }
        }
    }
    return best;
}

template <class Format, int TA, int TB, bool PAIR, class Epilogue>
int launch_form(const CUtensorMap& a, const CUtensorMap& b, Problem p, const typename Epilogue::Args& ep, int splits, int sm_count, cudaStream_t s) {
    using C = Cfg<TA, TB, PAIR>;
    auto kernel = plane_gemm_kernel<Format, TA, TB, PAIR, Epilogue>;
    static std::atomic<unsigned long long> opted{0};  // devices whose shared-memory limit has been raised for this kernel
    int dev = 0;
    CAKE_CUDA_OK(cudaGetDevice(&dev));
    if (dev >= 64 || !(opted.load() >> dev & 1)) {
        CAKE_CUDA_OK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM));
        if (dev < 64) opted |= 1ull << dev;
    }
    p.tiles_m = (p.rows + C::TILE_M - 1) / C::TILE_M;
    p.tiles_n = (p.cols + C::BN - 1) / C::BN;
    p.splits = splits;
    const long long tiles = p.symmetric ? (long long) p.tiles_m * (p.tiles_m + 1) / 2 : (long long) p.tiles_m * p.tiles_n;
    if (tiles * p.batch > (1LL << 27)) {
        set_error("the product has too many tiles");
        return CAKEB200_ERR_TOO_LARGE;
    }
    p.tiles = (int) tiles;
    const int per_tile = (PAIR ? 2 : 1) * splits;
    const int units = splits > 1 ? (int) (tiles * p.batch) : (int) std::min<long long>(tiles * p.batch, sm_count / per_tile);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned) (units * per_tile));
    cfg.blockDim = dim3(THREADS);
    cfg.dynamicSmemBytes = C::SMEM;
    cfg.stream = s;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned) per_tile;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    CAKE_CUDA_OK(cudaLaunchKernelEx(&cfg, kernel, a, b, p, ep));
    return CAKEB200_OK;
}

template <class Format, int TA, int TB, class Epilogue>
int launch(const CUtensorMap& a, const CUtensorMap& b, const Problem& p, const typename Epilogue::Args& ep, int sm_count, cudaStream_t s) {
    const Form f = pick_form(p.rows, p.cols, p.K, p.batch, p.symmetric != 0, sm_count);
    if (f.pair) return launch_form<Format, TA, TB, true, Epilogue>(a, b, p, ep, f.splits, sm_count, s);
    return launch_form<Format, TA, TB, false, Epilogue>(a, b, p, ep, f.splits, sm_count, s);
}

}  // namespace plane
}  // namespace cakeb200
