// Matrix product on the 5th-generation tensor cores for operands kept as sums of 16-bit planes.
//
// A value v is held as v = v0 + f v1 (+ f^2 v2), each term a 16-bit number that rounds what the terms before it left.
//   Fp16Planes: f = 2^-11, so that the second term has the range of the first; two terms carry 22 bits and a sign.  Absolute
//       resolution 2^-36, for data whose scale is known (below 2^16).
//   Bf16Planes: f = 1 and the range of FP32; two terms carry 16 bits and a sign, three all 24 bits of an FP32.
// With operands A (rows x K, TA planes) and B (cols x K, TB planes)
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
// An operand need not be stored with K along its rows.  Where it lies transposed in memory (K down the rows), boxes of 64 of K x
// 64 of its rows are loaded as they are and the MMA is told that the operand is "MN-major"; 16-bit types allow either.
// This is a choice per K block (Operand::turn), so that a symmetric matrix needs only the tiles on and below its diagonal
// in memory: a row of it is read along the row up to the diagonal and down the column from there.
//
// Two forms of one source, as in the FP32 product (sgemm_tf32x3.cu): PAIR = two CTAs on one 256 x 256 tile with
// tcgen05.mma.cta_group::2 (each stages its 128 rows of A and half of the tile's rows of B), else one CTA per 128 x 128
// tile.  A 128 x 128 x 16 MMA reads 8 KB of shared memory in its 64 clocks, all an SM delivers, and TMA writes come on
// top: with two planes a K block of 64 takes 1280 clocks at best.  A pair's 256 x 256 x 16 takes 128 clocks for the same
// 8 KB per SM: 1536 clocks per K block for twice the work per SM.
//
// Warp 0 issues TMA loads, warp 1 the MMAs, warp groups 1 and 2 fold and run the epilogue, a class with
//     struct Args;                                              // passed by value to the kernel
//     static __device__ void block(const Args&, const TileAt&, const float* v, uint32_t* patch, int lane);
// called by a warp for every 32 x 32 block of D: lane l holds row l of it in v[32], and patch[32][PATCH_LD] is the warp's own
// shared memory.
//
// The parts of a CTA are in Engine, from which kernels are put together: the plain product below, and the persistent kernel
// of orthogonalize.cu that runs a chain of products.
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
constexpr int BOX_BYTES = 64 * 64 * 2;     // 64 rows of 64 values
constexpr int PLANE_BYTES = 2 * BOX_BYTES; // one plane of one operand per stage and CTA: 128 rows of the operand in either form
constexpr int MAX_SMEM = 232448;
constexpr int PATCH_FLOATS = 32 * PATCH_LD;

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
};

// How a product (or `batch` products of one shape) is dealt to units, a unit being a CTA or a pair.  Tiles go to the units in
// turn; the tiles of a ragged last round, fewer than there are units, may be cut along K into `splits` parts of one unit
// each, which go to memory as FP32 and are joined afterwards, 32 x 32 blocks dealt out to all warps of the machine.
struct Tiling {
    int rows, cols, K;
    int symmetric;               // rows == cols and D = D^T: only tiles on and below the diagonal are computed
    int tiles_m, tiles_n, tiles; // tiles: of one product
    int whole;                   // tiles of all products that a unit finishes by itself
    int cut, splits;             // how many others there are, and into how many parts each is cut (cut * splits <= units)
};
struct Item {
    int tile, kb0, kb1, slot;    // slot < 0: whole K, straight to the epilogue
};
__device__ __forceinline__ bool item_at(const Tiling& g, int i, int unit, int units, Item& w) {
    const int blocks = (g.K + BK - 1) / BK;
    const int mine = (g.whole - unit + units - 1) / units;  // whole tiles of this unit
    if (i < mine) {
        w.tile = unit + i * units; w.kb0 = 0; w.kb1 = blocks; w.slot = -1;
        return true;
    }
    if (i > mine || unit >= g.cut * g.splits) return false;
    const int part = unit / g.cut;   // units next to one another read the same range of K
    w.tile = g.whole + unit % g.cut;
    w.kb0 = (int) ((long long) blocks * part / g.splits);
    w.kb1 = (int) ((long long) blocks * (part + 1) / g.splits);
    w.slot = unit;
    return true;
}
// tile `id` of a symmetric product's lower triangle, row by row
__device__ __forceinline__ void triangle(int id, int& tm, int& tn) {
    tm = (int) ((sqrtf(8.f * (float) id + 1.f) - 1.f) * 0.5f);
    while ((tm + 1) * (tm + 2) / 2 <= id) tm++;
    while (tm * (tm + 1) / 2 > id) tm--;
    tn = id - tm * (tm + 1) / 2;
}
__device__ __forceinline__ void place(const Tiling& g, int id, int& batch, int& tm, int& tn) {
    batch = id / g.tiles;
    const int t = id - batch * g.tiles;
    if (g.symmetric) triangle(t, tm, tn);
    else tile_coords(t, g.tiles_m, g.tiles_n, CAKEB200_SCHED_MKN, 8, tm, tn);
}

struct Problem {
    Tiling t;
    int batch;
    int a_turn, b_turn;  // ALONG or DOWN
    int chunk;           // K blocks between folds of `main`
    float* parts;        // of cut tiles: [slot][32 x 32 block][1024]
    int* status_word;
};

// D = F32, A and B of one 16-bit format, both K-major (bits 15 and 16 make A and B MN-major)
__host__ __device__ constexpr uint32_t idesc_16(uint32_t format, int m, int n) {
    return (1u << 4) | (format << 7) | (format << 10) | ((uint32_t) (n >> 3) << 17) | ((uint32_t) (m >> 4) << 24);
}

// 128-byte swizzled boxes of 64 rows.  K-major: a row of the box is a row of the operand, 8-row groups 1024 bytes apart, 16 of
// K are 32 bytes.  MN-major: a row of the box is one k of 64 rows of the operand, 8 of K are 1024 bytes apart (stride
// offset), the next 64 rows of the operand a box further (leading offset), 16 of K are 2048 bytes.
__device__ __forceinline__ uint64_t box_desc(uint32_t smem_addr, bool mn_major) {
    return make_kmajor_sw128_desc(smem_addr) + (mn_major ? (uint64_t) ((BOX_BYTES >> 4) - 1) << 16 : 0);
}

// How one operand of a product is read: `rows` of it from `row` on.  Of the K blocks before `turn` the operand's rows lie along the
// rows of memory, from there on along its columns.
struct Operand {
    const CUtensorMap* map;   // two: boxes of 128 rows for reading along the rows, then boxes of 64 for reading down
    int row, turn;
};
constexpr int ALONG = 1 << 30, DOWN = 0;  // values of `turn`: never, always
struct OperandMaps {
    CUtensorMap m[2];
};

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

// A block as 4 KB of FP32 in memory, row by row per lane and 16 bytes of every lane next to one another: whole lines both ways.
__device__ __forceinline__ void store_values(float* at, const float* v, int lane) {
#pragma unroll
    for (int q = 0; q < 8; q++) *reinterpret_cast<float4*>(at + q * 128 + lane * 4) = make_float4(v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]);
}
// from L2: another SM may have written it in this kernel
__device__ __forceinline__ void load_values(const float* at, float* v, int lane) {
#pragma unroll
    for (int q = 0; q < 8; q++) {
        const float4 u = __ldcg(reinterpret_cast<const float4*>(at + q * 128 + lane * 4));
        v[4 * q] = u.x; v[4 * q + 1] = u.y; v[4 * q + 2] = u.z; v[4 * q + 3] = u.w;
    }
}

// The sum of a block's parts, in part order: block b of `total` cut blocks.
__device__ __forceinline__ void join_parts(const float* parts, int b, int total, int splits, float* v, int lane) {
    load_values(parts + (long long) b * 1024, v, lane);
    for (int s = 1; s < splits; s++) {
        float u[32];
        load_values(parts + ((long long) s * total + b) * 1024, u, lane);
#pragma unroll
        for (int j = 0; j < 32; j++) v[j] += u[j];
    }
}

// What truncation takes from a sum, where that has a sign: `each` of it for every addition but the first `but`.
struct Loss {
    float each;
    int but;
    // what makes up for it in a sum over `depth` values
    __device__ __forceinline__ float factor(int depth) const { return 1.f + each * (float) ((depth + UMMA_K - 1) / UMMA_K - but); }
};

// What a CTA's roles share.  Every role walks the same sequence of (tile, K range) items and keeps its own place in it.
template <class Format, int TA, int TB, bool PAIR>
struct Engine {
    using C = Cfg<TA, TB, PAIR>;
    static constexpr int STAGES = C::STAGES, BN = C::BN, COLS = C::COLS;

    uint8_t* tiles;
    float* patch;             // of this drain warp
    uint32_t bar0, tmem_main, tmem_cross;
    volatile int* abort_flag;
    int* status_word;
    int warp, lane;
    uint32_t rank;            // within the pair: the even CTA issues the MMAs
    int stage;
    uint32_t phase, fold_phase, tile_phase;

    __device__ __forceinline__ uint32_t full_bar(int s) const { return bar0 + 8u * s; }
    __device__ __forceinline__ uint32_t empty_bar(int s) const { return bar0 + 8u * (STAGES + s); }
    __device__ __forceinline__ uint32_t main_full() const { return bar0 + 8u * (2 * STAGES); }
    __device__ __forceinline__ uint32_t main_empty() const { return bar0 + 8u * (2 * STAGES + 1); }
    __device__ __forceinline__ uint32_t cross_empty() const { return bar0 + 8u * (2 * STAGES + 2); }

    // All threads of the CTA (of both CTAs of a pair).
    __device__ __forceinline__ void open(uint8_t* smem_raw, int* status) {
        tiles = (uint8_t*) (((uintptr_t) smem_raw + 1023) & ~(uintptr_t) 1023);  // swizzled tiles: 1024-byte aligned
        uint64_t* bars = (uint64_t*) (tiles + STAGES * C::STAGE_BYTES);
        uint32_t* tmem_slot = (uint32_t*) (bars + 2 * STAGES + 3);
        abort_flag = (volatile int*) (tmem_slot + 1);
        status_word = status;
        warp = threadIdx.x >> 5;
        lane = threadIdx.x & 31;
        rank = PAIR ? cluster_ctarank() : 0u;
        patch = (float*) (tiles + STAGES * C::STAGE_BYTES + 256) + (warp & 7) * PATCH_FLOATS;
        bar0 = smem_u32(bars);
        stage = 0;
        phase = fold_phase = tile_phase = 0;
        if (threadIdx.x == 0) {
            for (int s = 0; s < STAGES; s++) {
                mbar_init(full_bar(s), 1);
                mbar_init(empty_bar(s), 1);
            }
            mbar_init(main_full(), 1);
            mbar_init(main_empty(), (PAIR ? 2 : 1) * DRAIN_WARPS);  // one arrival per drain warp (of both CTAs of a pair)
            mbar_init(cross_empty(), (PAIR ? 2 : 1) * DRAIN_WARPS);
            *abort_flag = 0;
            asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        }
        if (warp == 1) tmem_alloc<PAIR>(smem_u32(tmem_slot), (uint32_t) C::TMEM_COLS);
        tcgen05_fence_before();
        sync_all_t<PAIR>();
        tcgen05_fence_after();
        tmem_main = *tmem_slot;
        tmem_cross = tmem_main + (uint32_t) BN;
    }
    // All threads: nobody frees tensor memory or leaves while the other CTA of its pair may still touch it.
    __device__ __forceinline__ void close() {
        tcgen05_fence_before();
        sync_all_t<PAIR>();
        if (warp == 1) {
            tcgen05_fence_after();
            tmem_free<PAIR>(tmem_main, (uint32_t) C::TMEM_COLS);
        }
    }

    // TMA thread: K blocks [kb0, kb1) of this CTA's 128 rows of both operands; plane t of product `batch` lies at z = t * batches + batch.
    __device__ __forceinline__ void load_operand(const Operand& o, uint32_t base, int kb, int z, uint32_t bar) {
        if (kb < o.turn) {
            load_box<PAIR>(base, o.map, kb * BK, o.row, z, bar);
        } else {
            load_box<PAIR>(base, o.map + 1, o.row, kb * BK, z, bar);
            load_box<PAIR>(base + BOX_BYTES, o.map + 1, o.row + 64, kb * BK, z, bar);
        }
    }
    __device__ __forceinline__ bool load(const Operand& a, const Operand& b, int batch, int batches, int kb0, int kb1) {
        for (int kb = kb0; kb < kb1; kb++) {
            if (!mbar_wait(empty_bar(stage), phase ^ 1, abort_flag, status_word, 500 + stage)) return false;
            const uint32_t base = smem_u32(tiles + stage * C::STAGE_BYTES);
            if (rank == 0) mbar_expect_tx(full_bar(stage), (PAIR ? 2 : 1) * C::STAGE_BYTES);
#pragma unroll
            for (int i = 0; i < TA; i++) load_operand(a, base + i * PLANE_BYTES, kb, i * batches + batch, full_bar(stage));
#pragma unroll
            for (int j = 0; j < TB; j++) load_operand(b, base + (TA + j) * PLANE_BYTES, kb, j * batches + batch, full_bar(stage));
            if (++stage == STAGES) { stage = 0; phase ^= 1; }
        }
        return true;
    }
    // TMA thread that has issued everything: waits until it has been multiplied, so that no load is on its way into a CTA that has gone.
    __device__ __forceinline__ bool loads_done() {
        for (int s = 0; s < STAGES; s++) {
            if (!mbar_wait(empty_bar(stage), phase ^ 1, abort_flag, status_word, 505)) return false;
            if (++stage == STAGES) { stage = 0; phase ^= 1; }
        }
        return true;
    }
    // TMA thread that gave up: lets the loads already issued land before the CTA goes away (bounded).
    __device__ __forceinline__ void drain_loads() {
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

    // MMA thread (of the even CTA): the products of those K blocks, handed over every `chunk` blocks.
    __device__ __forceinline__ bool multiply(int a_turn, int b_turn, int kb0, int kb1, int chunk) {
        if (!mbar_wait(cross_empty(), tile_phase ^ 1, abort_flag, status_word, 510)) return false;
        tile_phase ^= 1;
        tcgen05_fence_after();
        uint32_t cross_acc = 0, main_acc = 0;
        int in_chunk = 0;
        for (int kb = kb0; kb < kb1; kb++) {
            if (!mbar_wait(full_bar(stage), phase, abort_flag, status_word, 520 + stage)) return false;
            tcgen05_fence_after();
            const uint32_t base = smem_u32(tiles + stage * C::STAGE_BYTES);
            const bool a_mn = kb >= a_turn, b_mn = kb >= b_turn;
            const uint32_t idesc = idesc_16(Format::FORMAT, C::TILE_M, BN) | (a_mn ? 1u << 15 : 0u) | (b_mn ? 1u << 16 : 0u);
            const uint64_t a0 = box_desc(base, a_mn), b0 = box_desc(base + TA * PLANE_BYTES, b_mn);
            const uint32_t a_step = a_mn ? 2048 >> 4 : 32 >> 4, b_step = b_mn ? 2048 >> 4 : 32 >> 4;  // 16 of K, in 16-byte units
#pragma unroll
            for (int k = 0; k < BK / UMMA_K; k++) {
#pragma unroll
                for (int s = C::LIMIT - 1; s > 0; s--)  // smallest products first
#pragma unroll
                    for (int i = 0; i < TA; i++) {
                        const int j = s - i;
                        if (j < 0 || j >= TB) continue;
                        umma<PAIR>(tmem_cross, a0 + (uint64_t) (i * (PLANE_BYTES >> 4) + k * a_step), b0 + (uint64_t) (j * (PLANE_BYTES >> 4) + k * b_step),
                                   idesc, cross_acc);
                        cross_acc = 1;
                    }
            }
            if (in_chunk == 0) {  // `main` starts from zero: its last fold has been read out
                if (!mbar_wait(main_empty(), fold_phase ^ 1, abort_flag, status_word, 530)) return false;
                fold_phase ^= 1;
                tcgen05_fence_after();
                main_acc = 0;
            }
#pragma unroll
            for (int k = 0; k < BK / UMMA_K; k++) {
                umma<PAIR>(tmem_main, a0 + (uint64_t) (k * a_step), b0 + (uint64_t) (k * b_step), idesc, main_acc);
                main_acc = 1;
            }
            umma_commit_t<PAIR>(empty_bar(stage));
            if (++stage == STAGES) { stage = 0; phase ^= 1; }
            if (++in_chunk == chunk || kb + 1 == kb1) {
                umma_commit_t<PAIR>(main_full());
                in_chunk = 0;
            }
        }
        return true;
    }

    // Drain warps: the sums of those K blocks (of a product over K), this warp's 32 rows x COLS columns, a row per lane.  A warp may only touch lanes
    // [32 * (warp % 4), +32) of tensor memory, so two warps share a quarter of the rows and take half of the columns each.
    __device__ __forceinline__ int quarter() const { return warp & 3; }
    __device__ __forceinline__ int half() const { return (warp - 4) >> 2; }
    __device__ __forceinline__ bool collect(int kb0, int kb1, int chunk, int K, const Loss& loss, float (&sum)[COLS]) {
        const uint32_t at = ((uint32_t) (quarter() * 32) << 16) + (uint32_t) (half() * COLS);
        float v[64];
#pragma unroll
        for (int j = 0; j < COLS; j++) sum[j] = 0.f;
        for (int kb = kb0; kb < kb1; kb += chunk) {
            bool ok = mbar_wait_for(main_full(), fold_phase, abort_flag, status_word, 540, WAIT_LIMIT_NS, 32);
            if (!__all_sync(0xffffffffu, ok)) return false;  // the tensor-memory loads below need the whole warp
            fold_phase ^= 1;
            tcgen05_fence_after();
            const float up = loss.factor(min(min(chunk, kb1 - kb) * BK, K - kb * BK));
#pragma unroll
            for (int c = 0; c < COLS; c += 64) {
                tmem_ld64(tmem_main + at + (uint32_t) c, v);
                tmem_ld_wait();
#pragma unroll
                for (int j = 0; j < 64; j++) sum[c + j] = fmaf(v[j], up, sum[c + j]);
            }
            tcgen05_fence_before();
            if (lane == 0) mbar_arrive_t<PAIR>(main_empty());
        }
        if (C::LIMIT > 1) {  // the commit of the last chunk covers the cross products too
#pragma unroll
            for (int c = 0; c < COLS; c += 64) {
                tmem_ld64(tmem_cross + at + (uint32_t) c, v);
                tmem_ld_wait();
#pragma unroll
                for (int j = 0; j < 64; j++) sum[c + j] = fmaf(v[j], 1.f / Format::TERM, sum[c + j]);
            }
            tcgen05_fence_before();
        }
        if (lane == 0) mbar_arrive_t<PAIR>(cross_empty());
        return true;
    }
    // f(column, row of 32 values) for each 32 x 32 block of this warp.  Rolled, the sums moving down by 32 registers a turn, so
    // that the code of a block exists once: unrolled four times it would run straight through from a cold instruction cache.
    template <typename F>
    __device__ __forceinline__ void blocks(float (&sum)[COLS], F f) {
#pragma unroll 1
        for (int c = 0; c < COLS; c += 32) {
            f(half() * COLS + c, sum);
#pragma unroll
            for (int j = 0; j + 32 < COLS; j++) sum[j] = sum[j + 32];
            __syncwarp();
        }
    }
};

// Registers follow the roles: 384 x 168 at launch = 128 x 40 + 256 x 232.
__device__ __forceinline__ void few_registers() { asm volatile("setmaxnreg.dec.sync.aligned.u32 40;"); }
__device__ __forceinline__ void many_registers() { asm volatile("setmaxnreg.inc.sync.aligned.u32 232;"); }

template <class Format, int TA, int TB, bool PAIR, class Epilogue>
__global__ void __launch_bounds__(THREADS, 1)
plane_gemm_kernel(const __grid_constant__ OperandMaps map_a, const __grid_constant__ OperandMaps map_b, const __grid_constant__ Problem p,
                  const __grid_constant__ typename Epilogue::Args ep) {
    using C = Cfg<TA, TB, PAIR>;
    extern __shared__ uint8_t smem_raw[];
    Engine<Format, TA, TB, PAIR> e;
    e.open(smem_raw, p.status_word);
    wait_for_previous_kernel();
    const int unit = (int) blockIdx.x / (PAIR ? 2 : 1), units = (int) gridDim.x / (PAIR ? 2 : 1);
    constexpr int WIDE = C::BN / 32, PER_TILE = (C::TILE_M / 32) * WIDE;  // 32 x 32 blocks of a tile, row by row
    Item w;
    int batch, tm, tn;
    if (e.warp < 4) {
        few_registers();
        if (e.warp == 0 && e.lane == 0) {
            bool ok = true;
            for (int k = 0; ok && item_at(p.t, k, unit, units, w); k++) {
                place(p.t, w.tile, batch, tm, tn);
                const Operand a = {map_a.m, tm * C::TILE_M + (int) e.rank * 128, p.a_turn}, b = {map_b.m, tn * C::BN + (int) e.rank * 128, p.b_turn};
                ok = e.load(a, b, batch, p.batch, w.kb0, w.kb1);
            }
            if (!ok || !e.loads_done()) e.drain_loads();
        } else if (e.warp == 1 && e.lane == 0 && e.rank == 0) {
            for (int k = 0; item_at(p.t, k, unit, units, w); k++)
                if (!e.multiply(p.a_turn, p.b_turn, w.kb0, w.kb1, p.chunk)) break;
        }
    } else {
        many_registers();
        float sum[C::COLS];
        for (int k = 0; item_at(p.t, k, unit, units, w); k++) {
            if (!e.collect(w.kb0, w.kb1, p.chunk, p.t.K, Loss{0.f, 0}, sum)) break;
            TileAt at;
            place(p.t, w.tile, at.batch, tm, tn);
            const int row = (int) e.rank * BM + e.quarter() * 32;
            at.row = tm * C::TILE_M + row;
            e.blocks(sum, [&](int column, const float* v) {
                at.col = tn * C::BN + column;
                if (w.slot >= 0) store_values(p.parts + ((long long) w.slot * PER_TILE + row / 32 * WIDE + column / 32) * 1024, v, e.lane);
                else if (at.row < p.t.rows && at.col < p.t.cols) Epilogue::block(ep, at, v, (uint32_t*) e.patch, e.lane);
            });
        }
    }
    e.close();
}

// The epilogue of the cut tiles of a plane_gemm_kernel of that form: a warp per 32 x 32 block.
template <bool PAIR, class Epilogue>
__global__ void __launch_bounds__(256)
join_kernel(const __grid_constant__ Problem p, const __grid_constant__ typename Epilogue::Args ep) {
    constexpr int SIDE = PAIR ? 256 : 128, WIDE = SIDE / 32, PER_TILE = WIDE * WIDE;
    __shared__ uint32_t patches[8][PATCH_FLOATS];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int total = p.t.cut * PER_TILE, b = (int) blockIdx.x * 8 + warp;
    wait_for_previous_kernel();
    if (b >= total) return;
    TileAt at;
    int tm, tn;
    place(p.t, p.t.whole + b / PER_TILE, at.batch, tm, tn);
    at.row = tm * SIDE + b % PER_TILE / WIDE * 32;
    at.col = tn * SIDE + b % WIDE * 32;
    if (at.row >= p.t.rows || at.col >= p.t.cols) return;
    float v[32];
    join_parts(p.parts, b, total, p.t.splits, v, lane);
    Epilogue::block(ep, at, v, patches[warp], lane);
}

// ------------------------------------------------------------------ epilogue helpers

// Planes of a matrix in memory: element (r, c) of term t of product `batch` at base + ((t * batches + batch) * rows + r) * ld + c,
// ld a multiple of 8.
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
// Eight consecutive values of two planes, as FP32; from L2, as another SM may have written them in this kernel.
template <class Format>
__device__ __forceinline__ void load8(const Planes& p, int batch, int r, int c, float* v) {
    const uint16_t* at = p.base + ((long long) batch * p.rows + r) * p.ld + c;
    const uint4 h = __ldcg(reinterpret_cast<const uint4*>(at)), l = __ldcg(reinterpret_cast<const uint4*>(at + (long long) p.batches * p.rows * p.ld));
    const uint32_t hi[4] = {h.x, h.y, h.z, h.w}, lo[4] = {l.x, l.y, l.z, l.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float2 a = Format::value(hi[i]), b = Format::value(lo[i]);
        v[2 * i] = fmaf(b.x, 1.f / Format::TERM, a.x);
        v[2 * i + 1] = fmaf(b.y, 1.f / Format::TERM, a.y);
    }
}

// A block through the patch to four lanes per row: f(row of the block, column of the block, eight values from there on), eight rows
// at a time.  A store costs the SM a clock for every row that it touches, so whole rows are what it should see.
template <typename F>
__device__ __forceinline__ void by_eights(const float* v, uint32_t* patch, int lane, F f) {
#pragma unroll
    for (int j = 0; j < 32; j++) patch[lane * PATCH_LD + j] = __float_as_uint(v[j]);
    __syncwarp();
#pragma unroll
    for (int q = 0; q < 4; q++) {
        const int r = 8 * q + (lane >> 2), c = 8 * (lane & 3);
        float u[8];
#pragma unroll
        for (int e = 0; e < 8; e++) u[e] = __uint_as_float(patch[r * PATCH_LD + c + e]);
        f(r, c, u);
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

inline int padded(int cols) { return (cols + 7) / 8 * 8; }  // rows start on 16-byte boundaries, as TMA wants them
inline size_t plane_bytes(int terms, int batches, int rows, int cols) {
    return ((size_t) terms * batches * rows * padded(cols) * 2 + 1023) / 1024 * 1024;
}
// the two tensor maps of an operand over planes: boxes of 128 and of 64 rows, 64 values each
template <class Format>
int encode_planes(CUtensorMap* maps, const Planes& p, int terms) {
    const unsigned long long dims[3] = {(unsigned long long) p.cols, (unsigned long long) p.rows, (unsigned long long) terms * p.batches};
    const unsigned long long strides[2] = {(unsigned long long) p.ld * 2, (unsigned long long) p.ld * 2 * p.rows};
    const unsigned along[3] = {64, 128, 1}, down[3] = {64, 64, 1};
    const int rc = encode_tiled_16(&maps[0], Format::FORMAT == 1, p.base, 3, dims, strides, along, true);
    return rc ? rc : encode_tiled_16(&maps[1], Format::FORMAT == 1, p.base, 3, dims, strides, down, true);
}

inline long long count_tiles(int rows, int cols, int batch, bool symmetric, int side) {
    const long long m = (rows + side - 1) / side, n = (cols + side - 1) / side;
    return batch * (symmetric ? m * (m + 1) / 2 : m * n);
}

// What the model below knows about a kernel, in microseconds: measured with globaltimer stamps.
struct Costs {
    double block[2];   // a K block, [0] on a single SM, [1] on a pair
    double between;    // from the last store of a part to the first load of a part, and likewise to what follows the product
};
// A K block: the MMAs (64 and 128 clocks each) or the shared-memory traffic (16 KB per plane written, 8 KB per MMA read, 128 bytes
// a clock), whichever is longer, at 1.85 GHz and with the 10 % that both lose in practice (three products of two planes:
// 0.75 and 0.93 measured); or its way from L2, 47 bytes a clock at best (measured on products of one plane, four stages as well as six),
// which decides for one plane against two on single SMs.  500 x 4096 x 4096 in BF16 takes 51 us on pairs, 59 on single SMs; 65 x 4096
// x 4096 41 and 37; in every shape of 65 to 2000 rows and 2048^2 to 16384 x 8192 weights that was timed the faster form is chosen.
inline Costs costs_of(int ta, int tb, int products, double between) {
    const double load = (ta + tb) * 16384.0 / 47.0 / 1.1, smem = std::max(load, ((ta + tb) * 16384.0 + products * 4 * 8192.0) / 128.0);
    Costs c;
    c.block[0] = std::max(smem, products * 4 * 64.0) * 1.1 / 1850;
    c.block[1] = std::max(smem, products * 4 * 128.0) * 1.1 / 1850;
    c.between = between;
    return c;
}

// Deals a product to `units` units of one form and returns its time by the model: 2 to the first MMA, 0.7 to read a tile's sums
// out, 2.0 and 1.0 per 32 x 32 block of a warp, four of a pair's tile and two of a single one's; where parts are stored 1.0
// and 0.7 instead, then 2.4 and 0.15 per part for each block that a warp joins.
inline double plan(Tiling* g, int rows, int cols, int K, int symmetric, int batch, bool pair, int units, const Costs& costs, bool may_cut = true) {
    const int side = pair ? 256 : 128, blocks = (K + BK - 1) / BK;
    g->rows = rows; g->cols = cols; g->K = K; g->symmetric = symmetric;
    g->tiles_m = (rows + side - 1) / side;
    g->tiles_n = (cols + side - 1) / side;
    g->tiles = symmetric ? g->tiles_m * (g->tiles_m + 1) / 2 : g->tiles_m * g->tiles_n;
    const int total = g->tiles * batch, left = total % units, rounds = total / units;
    const double block_time = costs.block[pair ? 1 : 0], round_time = blocks * block_time + 0.7;
    g->whole = total; g->cut = 0; g->splits = 1;
    double best = (rounds + (left ? 1 : 0)) * round_time + 2 + (pair ? 8 : 2) + costs.between;
    const int forced = option_get(OPT_K_PIECES);
    if (left == 0 || forced == 1 || !may_cut) return best;
    for (int splits = 1; splits <= std::min(units / left, blocks); splits++) {
        const int warps = units * (pair ? 2 : 1) * DRAIN_WARPS, per_warp = (left * (side / 32) * (side / 32) + warps - 1) / warps;
        const double time = rounds * round_time + (blocks + splits - 1) / splits * block_time + 0.7 + 2 + (pair ? 4 : 1.4) + costs.between +
                            per_warp * (2.4 + 0.15 * splits) + costs.between;
        if (forced ? splits <= forced : time < best) {
            g->whole = total - left; g->cut = left; g->splits = splits;
            best = time;
        }
    }
    return best;
}

constexpr int MAX_UNITS = 160;  // single SMs; half as many pairs
inline int units_of(bool pair, int sm_count) { return std::min(pair ? sm_count / 2 : sm_count, pair ? MAX_UNITS / 2 : MAX_UNITS); }
// Room for the parts of `pieces` pieces (K blocks of all tiles) at most, whatever the number of SMs: a part is a tile of one form.
inline size_t parts_bytes(long long pieces, bool pair) {
    return (size_t) std::min<long long>(pieces, pair ? MAX_UNITS / 2 : MAX_UNITS) * (pair ? 256 * 256 * 4 : 128 * 128 * 4);
}

template <typename... P>
int launch_kernel(void (*kernel)(P...), unsigned grid, unsigned threads, unsigned cluster, size_t smem, cudaStream_t s, P... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = cluster;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = cluster > 1 ? 2 : 1;
    CAKE_CUDA_OK(cudaLaunchKernelEx(&cfg, kernel, args...));
    return CAKEB200_OK;
}

template <class Format, int TA, int TB, bool PAIR, class Epilogue>
int launch_form(const OperandMaps& a, const OperandMaps& b, const Problem& p, const typename Epilogue::Args& ep, int units, cudaStream_t s) {
    using C = Cfg<TA, TB, PAIR>;
    auto kernel = plane_gemm_kernel<Format, TA, TB, PAIR, Epilogue>;
    static std::atomic<unsigned long long> opted{0};  // devices whose shared-memory limit has been raised for this kernel
    int dev = 0;
    CAKE_CUDA_OK(cudaGetDevice(&dev));
    if (dev >= 64 || !(opted.load() >> dev & 1)) {
        CAKE_CUDA_OK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM));
        if (dev < 64) opted |= 1ull << dev;
    }
    units = std::min(units, std::max(p.t.whole, p.t.cut * p.t.splits));
    int rc = launch_kernel(kernel, (unsigned) (PAIR ? 2 * units : units), THREADS, PAIR ? 2u : 1u, C::SMEM, s, a, b, p, ep);
    if (rc || p.t.cut == 0) return rc;
    const unsigned blocks = (unsigned) (p.t.cut * (PAIR ? 64 : 16) + 7) / 8;
    return launch_kernel(join_kernel<PAIR, Epilogue>, blocks, 256u, 1u, 0, s, p, ep);
}

// One product (or p.batch of them).  `parts` of the problem holds parts_bytes(K blocks of all tiles) of the larger form; nullptr: no
// tile is cut.
template <class Format, int TA, int TB, int PRODUCTS, class Epilogue>
int launch(const OperandMaps& a, const OperandMaps& b, Problem p, int rows, int cols, int K, const typename Epilogue::Args& ep, int sm_count,
           cudaStream_t s, int* launches) {
    if (count_tiles(rows, cols, p.batch, false, 128) > (1LL << 27)) {
        set_error("the product has too many tiles");
        return CAKEB200_ERR_TOO_LARGE;
    }
    const Costs costs = costs_of(TA, TB, PRODUCTS, 3.0);
    const int forced = option_get(OPT_PAIR);  // 1: pairs, 2: single SMs, 0: the faster by the model
    Tiling single, pair;
    const double t_single = plan(&single, rows, cols, K, 0, p.batch, false, units_of(false, sm_count), costs, p.parts != nullptr);
    const double t_pair = plan(&pair, rows, cols, K, 0, p.batch, true, units_of(true, sm_count), costs, p.parts != nullptr);
    const bool paired = forced ? forced == 1 : t_pair < t_single;
    p.t = paired ? pair : single;
    if (launches) *launches += p.t.cut ? 2 : 1;
    if (paired) return launch_form<Format, TA, TB, true, Epilogue>(a, b, p, ep, units_of(true, sm_count), s);
    return launch_form<Format, TA, TB, false, Epilogue>(a, b, p, ep, units_of(false, sm_count), s);
}

}  // namespace plane
}  // namespace cakeb200
