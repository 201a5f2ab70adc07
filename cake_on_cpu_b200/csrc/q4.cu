// Products with weights held in 4 bits (the packed form is described in q4.cuh):
//     y[r, n] = sum_k x[r, k] w[n, k] (+ bias[n])        and its gradient for the input
//     dx[r, k] = sum_n dy[r, n] w[n, k].
//
// With few rows both are bound by reading the codes from HBM: half a byte per multiply-add and row.  What stands in
// the way of that bound is the work of turning codes into numbers.  At 6.4 TB/s an SM receives 46 codes per clock, so a
// lane may spend 2.8 instructions on one.  Converting a code to FP32 and multiplying takes about four; here a mask and a
// shift place a pair of codes in the mantissas of two 16-bit numbers, exactly, and mma.m16n8k16 multiplies 16 x 16 of them with
// up to eight rows of x at once.  The products are exact and summed in FP32; the sum of a group is multiplied by its scale
// in FP32 and added to the row's total, so scales are never rounded into the weights.  (tcgen05.mma would take the weights from shared memory: writing converted
// codes there costs four times the bytes that are read from HBM.)
// The numbers are 128 + q as BF16 or 1024 + q as FP16, the code in the last bits of the mantissa, and 128 + z or 1024 + z is
// subtracted from every pair right away, so that a product is w x / scale.  (Codes as subnormal FP16 and the zero point taken out of the
// group's sum with its sum of x would save the subtractions, 7.0 to 6.3 us at one row of 4096 x 4096; but then the error goes with
// the sum of |x| q: a large x under a weight of zero leaves its rounding in the result.)
// A 32-bit x goes through the 16-bit multiplier as three terms x = x0 + x1 + x2 of 8 mantissa bits each (truncations,
// so the split is exact and cannot overflow); their products are summed in FP32.
#include <algorithm>
#include <atomic>
#include <type_traits>

#include "q4.cuh"

namespace cakeb200 {
namespace {

constexpr int MAX_CLUSTER = 8;

// ------------------------------------------------------------------ small device helpers

template <typename M>
__device__ __forceinline__ void mma(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
    if constexpr (sizeof(M) == 2 && std::is_same<M, __half>::value)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// The power of two whose last mantissa bit counts 1, in both halves of a word: 128 as BF16, 1024 as FP16.
template <typename M> constexpr uint32_t POWER = std::is_same<M, __half>::value ? 0x64006400u : 0x43004300u;
// that power + z in both halves (z < 16)
template <typename M>
__device__ __forceinline__ uint32_t zero_pair(uint32_t z) { return POWER<M> | (z << 16) | z; }
// The four A registers of a word's MMA.  A code in the mantissa of that power, then the power and the zero point subtracted, both
// halves at once: exact whole numbers.  sub_lo / sub_hi: zero_pair of rows a / a + 8.
template <typename M>
__device__ __forceinline__ void unpack_centred(uint32_t w, uint32_t sub_lo, uint32_t sub_hi, uint32_t* a) {
    using M2 = typename std::conditional<std::is_same<M, __half>::value, __half2, __nv_bfloat162>::type;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const uint32_t v = ((w >> (4 * i)) & 0x000f000fu) | POWER<M>;
        const uint32_t sub = (i & 1) ? sub_hi : sub_lo;
        const M2 r = __hsub2(*reinterpret_cast<const M2*>(&v), *reinterpret_cast<const M2*>(&sub));
        a[i] = *reinterpret_cast<const uint32_t*>(&r);
    }
}

// The MMA's type and the number of terms of x, for the forward product.
template <typename T>
struct Codes {
    using M = typename std::conditional<std::is_same<T, __half>::value, __half, __nv_bfloat16>::type;
    static constexpr int TERMS = sizeof(T) == 4 ? 3 : 1;
};
// Codes are read once and go past L1 into a queue of the lane's own in shared memory, so that many are on their way without
// holding registers; a lane reads back what it asked for itself.
__device__ __forceinline__ void fetch16(uint4* to, const uint4* from) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t) __cvta_generic_to_shared(to)), "l"(from) : "memory");
}
__device__ __forceinline__ void fetch_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int LEFT>
__device__ __forceinline__ void fetch_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(LEFT) : "memory"); }

__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ float load_remote(const float* local, int rank) {
    uint32_t a = (uint32_t) __cvta_generic_to_shared(local), r;
    float v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(rank));
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(r) : "memory");
    return v;
}

// Hands the sums of `red`[SETS][E] over the sets of all CTAs of the cluster, in that fixed order, to `store(e, value)`: every CTA
// finishes its share of the E elements.
template <int E, int SETS, int WARPS, typename F>
__device__ __forceinline__ void join(const float* red, int rank, int cluster, F store) {
    const int per = E / cluster;
    for (int i = threadIdx.x; i < per; i += WARPS * 32) {
        const int e = rank * per + i;
        float s = 0.f;
        for (int c = 0; c < cluster; c++) {
#pragma unroll
            for (int w = 0; w < SETS; w++) s += load_remote(red + w * E + e, c);
        }
        store(e, s);
    }
}

// Whether the kernels below take a product, or the weights are expanded and multiplied on tcgen05 (q4_gemm.cu).  These read the codes
// again for every 32 (gradient: 16) rows, the others pay for three launches, a workspace and the expanded weights whatever the
// number of rows.  us here / there: y of 16-bit types, 128 rows, 4096 x 4096 41 / 41, 8192 x 4096 66 / 68, 16384 x 8192 184 / 248 (192
// rows 270 / 264), 2048 x 2048 20 / 25 (256 rows 29 / 27); 512 rows, 1024 x 1024 23 / 23.  FP32 takes three MMAs here: 65 rows, 4096 x
// 4096 59 / 53, 16384 x 8192 326 / 348, 128 rows 434 / 348; 1024 x 1024, 384 rows 29 / 29.  Gradients, 65 rows, 4096 x 4096 BF16 53 / 41,
// 2048 x 2048 25 / 25, 1024 x 1024, 192 rows 20 / 23, 256 rows 27 / 20.
bool few_rows(const Q4View& w, int rows, int type, bool dx) {
    if (rows <= 64) return true;
    if (rows > 1024 || option_get(OPT_PAIR) || option_get(OPT_K_PIECES)) return false;  // those options are about tcgen05 tiles
    if (rows <= 128 && type != CAKEB200_F32 && !dx) return true;
    return (long long) rows * w.N * w.K <= (dx ? 1LL << 28 : 1LL << 29);
}

struct Q4Args {
    Q4View w;
    const void* in;      // x (rows x K) or dy (rows x N)
    void* out;           // y (rows x N) or dx (rows x K)
    const void* bias;    // N elements of the input's type, or nullptr
    long long ld_in, ld_out;
    int rows;
    int vec;             // 16-byte loads of x allowed
    int cluster;
    int chunks;          // of 8 NT rows
};

// ------------------------------------------------------------------ y = x W^T + b

// B fragments of a lane for a block: features 32 h + 8 t + 0 .. 7, h = 0, 1, of its row, pairs of features to a register.  `x` points at
// the first of them; `inside`: 16-byte loads are allowed and the block ends within the row.
template <typename T>
__device__ __forceinline__ void load_x(const T* x, bool inside, int left, uint32_t (*b)[Codes<T>::TERMS]) {
    constexpr int TERMS = Codes<T>::TERMS;
#pragma unroll
    for (int h = 0; h < 2; h++) {
        const T* p = x + 32 * h;
        if constexpr (sizeof(T) == 2) {
            if (inside) {
                const uint4 v = __ldg(reinterpret_cast<const uint4*>(p));
                b[4 * h][0] = v.x; b[4 * h + 1][0] = v.y; b[4 * h + 2][0] = v.z; b[4 * h + 3][0] = v.w;
            } else {
                const uint16_t* u = reinterpret_cast<const uint16_t*>(p);
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const uint32_t lo = 32 * h + 2 * i < left ? __ldg(u + 2 * i) : 0, hi = 32 * h + 2 * i + 1 < left ? __ldg(u + 2 * i + 1) : 0;
                    b[4 * h + i][0] = lo | (hi << 16);
                }
            }
        } else {
            float v[8];
            if (inside) {
                const float4 u0 = __ldg(reinterpret_cast<const float4*>(p)), u1 = __ldg(reinterpret_cast<const float4*>(p) + 1);
                v[0] = u0.x; v[1] = u0.y; v[2] = u0.z; v[3] = u0.w; v[4] = u1.x; v[5] = u1.y; v[6] = u1.z; v[7] = u1.w;
            } else {
#pragma unroll
                for (int i = 0; i < 8; i++) v[i] = 32 * h + i < left ? __ldg(p + i) : 0.f;
            }
#pragma unroll
            for (int i = 0; i < 4; i++) split_pair<TERMS>(v[2 * i], v[2 * i + 1], b[4 * h + i]);
        }
    }
}

// Scales and zero points of rows a and a + 8 for one block row and step.
template <int GROUPS>
struct Scales {
    uint32_t scales[GROUPS];   // two to a word
    uint32_t zeros[(GROUPS + 1) / 2];
};
// `at`: block row times steps plus step.
template <int GROUPS>
__device__ __forceinline__ void load_scales(const Q4View& w, int at, int a, Scales<GROUPS>& s) {
    const long long place = (long long) at * (16 * GROUPS) + a * (2 * GROUPS);
    const uint16_t* p = w.scales + place;
    if constexpr (GROUPS == 1) {
        s.scales[0] = __ldg(reinterpret_cast<const uint32_t*>(p));
    } else if constexpr (GROUPS == 2) {
        const uint2 v = __ldg(reinterpret_cast<const uint2*>(p));
        s.scales[0] = v.x; s.scales[1] = v.y;
    } else {
        const uint4 v = __ldg(reinterpret_cast<const uint4*>(p));
        s.scales[0] = v.x; s.scales[1] = v.y; s.scales[2] = v.z; s.scales[3] = v.w;
    }
    if (w.zeros) {
        const uint8_t* z = w.zeros + place;
        if constexpr (GROUPS == 1) s.zeros[0] = __ldg(reinterpret_cast<const uint16_t*>(z));
        else if constexpr (GROUPS == 2) s.zeros[0] = __ldg(reinterpret_cast<const uint32_t*>(z));
        else {
            const uint2 v = __ldg(reinterpret_cast<const uint2*>(z));
            s.zeros[0] = v.x; s.zeros[1] = v.y;
        }
    } else {
#pragma unroll
        for (int i = 0; i < (GROUPS + 1) / 2; i++) s.zeros[i] = 0x08080808u;
    }
}

// An item is R block rows (16 R output features) x 8 NT rows of x.  Clusters take items in turn; the warps of a cluster share
// out an item's steps.  While a step is multiplied the codes of the next two and the scales of the next one are on their way,
// across the ends of items, and the sums of an item are joined while the next one is multiplied: warps leave them in shared
// memory, arrive at the cluster's barrier, and only wait for it at the end of the next item.  (With one CTA per item and
// the join at its end the machine stood a quarter idle: 512 items do not divide among 148 SMs.)
constexpr int AHEAD = 3;  // steps in a lane's queue

template <typename T, int NT, int R, int GROUPS, int WARPS>
__global__ void __launch_bounds__(WARPS * 32)
q4_linear_kernel(const Q4Args p) {
    using M = typename Codes<T>::M;
    constexpr int TERMS = Codes<T>::TERMS;
    constexpr int E = R * NT * 128;
    constexpr int QUEUE = AHEAD * R * 64;  // of a warp, in 16-byte pieces
    // with few columns there are registers for what keeps a lone warp busy: x of a whole step loaded at its start, and two chains of
    // dependent MMAs per sum.  FP32 takes the products with the leading terms of x apart from the others: an MMA truncates the sum
    // that it adds to, and 8 such additions per group of 128 instead of 24 leave a third of that
    constexpr int HALVES = NT == 1 && TERMS == 1 ? 2 : 1, CHAINS = NT == 1 || TERMS > 1 ? 2 : 1;
    extern __shared__ uint4 shared[];      // queues, then two sets of sums
    float* red = (float*) (shared + WARPS * QUEUE);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, a = lane >> 2, t = lane & 3;
    uint4* queue = shared + warp * QUEUE + lane;
    const int rank = (int) blockIdx.x % p.cluster, unit = (int) blockIdx.x / p.cluster, units = (int) gridDim.x / p.cluster;
    const int rbs = p.w.row_tiles / R, items = rbs * p.chunks;
    const int part = rank * WARPS + warp, parts = p.cluster * WARPS;
    const int s0 = (int) ((long long) p.w.steps * part / parts), s1 = (int) ((long long) p.w.steps * (part + 1) / parts);
    const int mine = s1 > s0 ? (items - unit + units - 1) / units * (s1 - s0) : 0;  // steps of this warp, over all its items

    // Steps in the order in which this warp does them; `at` of block row r is r * steps further.
    struct Cursor {
        int item, left, at;
    };
    auto place = [&](int item) { return item % rbs * R * p.w.steps + s0; };
    auto advance = [&](Cursor& c) {
        c.at++;
        if (--c.left == 0) {
            c.left = s1 - s0;
            c.item += units;
            c.at = place(c.item);
        }
    };
    auto fetch = [&](const Cursor& c, int where) {
#pragma unroll
        for (int r = 0; r < R; r++) {
            const uint4* from = p.w.codes + (long long) (c.at + r * p.w.steps) * 64 + lane;
            fetch16(queue + (where * R + r) * 64, from);
            fetch16(queue + (where * R + r) * 64 + 32, from + 32);
        }
    };
    Cursor codes_cursor = {unit, s1 - s0, place(unit)}, scales_cursor = codes_cursor;
    Scales<GROUPS> next[R];
#pragma unroll
    for (int i = 0; i < AHEAD - 1; i++) {
        if (i < mine) {
            fetch(codes_cursor, i);
            advance(codes_cursor);
        }
        fetch_commit();
    }
    if (mine) {
#pragma unroll
        for (int r = 0; r < R; r++) load_scales(p.w, scales_cursor.at + r * p.w.steps, a, next[r]);
        advance(scales_cursor);
    }

    T* out = (T*) p.out;
    const T* bias = (const T*) p.bias;
    auto finish = [&](int item, int set) {
        const int rb = item % rbs, row0 = item / rbs * 8 * NT;
        join<E, WARPS, WARPS>(red + set * WARPS * E, rank, p.cluster, [&](int e, float v) {
            const int l = e & 31, i = (e >> 5) & 3, nt = (e >> 7) % NT, r = (e >> 7) / NT;
            const int n = (rb * R + r) * 16 + (l >> 2) + (i >> 1) * 8, row = row0 + nt * 8 + (l & 3) * 2 + (i & 1);
            if (n >= p.w.N || row >= p.rows) return;
            if (bias) v += to_float(bias[n]);
            out[row * p.ld_out + n] = from_float<T>(v);
        });
    };

    int slot = 0, free = AHEAD - 1, done = 0, set = 0;
    for (int item = unit; item < items; item += units, set ^= 1) {
        const int row0 = item / rbs * 8 * NT;
        const T* x[NT];  // rows past the last repeat it; their columns of the MMA are not stored
#pragma unroll
        for (int nt = 0; nt < NT; nt++) x[nt] = (const T*) p.in + (long long) min(row0 + nt * 8 + a, p.rows - 1) * p.ld_in + s0 * 128 + t * 8;
        float total[R][NT][4] = {};
        for (int step = s0; step < s1; step++, done++) {
            Scales<GROUPS> now[R];
            const bool inside = p.vec && step * 128 + 128 <= p.w.K;
            uint32_t b[HALVES][NT][8][TERMS];
            auto load = [&](int half) {
#pragma unroll
                for (int nt = 0; nt < NT; nt++) {
                    load_x<T>(x[nt], inside, p.w.K - (step * 128 + half * 64 + t * 8), b[half % HALVES][nt]);
                    x[nt] += 64;
                }
            };
            if (HALVES == 2) { load(0); load(1); }
            if (done + AHEAD - 1 < mine) {
                fetch(codes_cursor, free);
                advance(codes_cursor);
            }
            fetch_commit();
#pragma unroll
            for (int r = 0; r < R; r++) now[r] = next[r];
            if (done + 1 < mine) {
#pragma unroll
                for (int r = 0; r < R; r++) load_scales(p.w, scales_cursor.at + r * p.w.steps, a, next[r]);
                advance(scales_cursor);
            }
            fetch_wait<AHEAD - 1>();
            float acc[R][NT][CHAINS][4];
#pragma unroll
            for (int half = 0; half < 2; half++) {  // a block of 64 features
                if (HALVES == 1) load(half);
#pragma unroll
                for (int part = 0; part < 2; part++) {  // 32 features, words 2 part and 2 part + 1
                    constexpr int PARTS = 4 / GROUPS;   // of a group
                    const int g = (half * 2 + part) / PARTS;
                    const bool first = (half * 2 + part) % PARTS == 0, last = (half * 2 + part) % PARTS == PARTS - 1;
                    if (first) {
#pragma unroll
                        for (int nt = 0; nt < NT; nt++) {
#pragma unroll
                            for (int i = 0; i < CHAINS * 4; i++) {
#pragma unroll
                                for (int r = 0; r < R; r++) acc[r][nt][i / 4][i % 4] = 0.f;
                            }
                        }
                    }
                    uint2 c[R];
#pragma unroll
                    for (int r = 0; r < R; r++) c[r] = reinterpret_cast<const uint2*>(&queue[(slot * R + r) * 64 + half * 32])[part];
#pragma unroll
                    for (int j = 2 * part; j < 2 * part + 2; j++) {
#pragma unroll
                        for (int r = 0; r < R; r++) {
                            const uint32_t z = now[r].zeros[g / 2] >> (16 * (g & 1));
                            uint32_t w[4];
                            unpack_centred<M>(j & 1 ? c[r].y : c[r].x, zero_pair<M>(z & 15u), zero_pair<M>((z >> 8) & 15u), w);
#pragma unroll
                            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                                for (int u = TERMS - 1; u >= 0; u--)
                                    mma<M>(acc[r][nt][TERMS > 1 ? u > 0 : j % CHAINS], w, b[half % HALVES][nt][2 * j][u], b[half % HALVES][nt][2 * j + 1][u]);
                        }
                    }
                    if (last) {  // the group is complete
#pragma unroll
                        for (int r = 0; r < R; r++) {
                            const float s_lo = q4_scale((uint16_t) now[r].scales[g], p.w.scale_bf16), s_hi = q4_scale((uint16_t) (now[r].scales[g] >> 16), p.w.scale_bf16);
#pragma unroll
                            for (int nt = 0; nt < NT; nt++) {
#pragma unroll
                                for (int i = 0; i < 2; i++) {
                                    float lo = acc[r][nt][0][i], hi = acc[r][nt][0][i + 2];
                                    if (CHAINS == 2) {
                                        lo += acc[r][nt][CHAINS - 1][i];
                                        hi += acc[r][nt][CHAINS - 1][i + 2];
                                    }
                                    total[r][nt][i] = fmaf(s_lo, lo, total[r][nt][i]);
                                    total[r][nt][i + 2] = fmaf(s_hi, hi, total[r][nt][i + 2]);
                                }
                            }
                        }
                    }
                }
            }
            free = slot;
            if (++slot == AHEAD) slot = 0;
        }
        if (item != unit) {  // the item before this one: everybody's sums of it are there
            cluster_wait();
            finish(item - units, set ^ 1);
        }
#pragma unroll
        for (int r = 0; r < R; r++)
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                for (int i = 0; i < 4; i++) red[(set * WARPS + warp) * E + ((r * NT + nt) * 4 + i) * 32 + lane] = total[r][nt][i];
        __syncwarp();
        cluster_arrive();
        if (item + units >= items) {
            cluster_wait();
            finish(item, set);
        }
    }
    cluster_arrive();  // nobody leaves while its sums may still be read
    cluster_wait();
}

// ------------------------------------------------------------------ dx = dy W

// 8 x 8 matrix of 16-bit elements, transposed across the warp
__device__ __forceinline__ uint32_t transpose8(uint32_t v) {
    uint32_t o;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(o) : "r"(v));
    return o;
}

// A CTA computes one k block (64 input features) x 8 NT rows; its warps share out the block rows of the CTA, the CTAs
// of a cluster those of the product.  The reduction runs over output features, whose scales differ, so the scale goes
// into the other operand: dy[r, n] s[n, g], formed in FP32 and split into TERMS bf16 terms (two for 16-bit types, each rounded
// to nearest: 2^-17 relative and of either sign, far below their own rounding; three for FP32, exactly).  Sums of one block row (16 n) leave the MMA for an FP32 total.
template <typename T, int NT, int GROUPS, int WARPS>
__global__ void __launch_bounds__(WARPS * 32)
q4_linear_dx_kernel(const Q4Args p) {
    using M = __nv_bfloat16;
    constexpr int TERMS = sizeof(T) == 4 ? 3 : 2;
    constexpr int E = NT * 512;
    constexpr int DX_AHEAD = 8;            // block rows in a lane's queue
    __shared__ uint4 shared[WARPS * (DX_AHEAD * 128 > E ? DX_AHEAD * 32 : E / 4)];
    float* red = (float*) shared;          // the queues' place, once they are empty
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, a = lane >> 2, t = lane & 3;
    uint4* queue = shared + warp * DX_AHEAD * 32 + lane;
    const int rank = (int) blockIdx.x % p.cluster, kb = (int) blockIdx.x / p.cluster;  // block of 64 features
    const int row0 = (int) blockIdx.y * 8 * NT;
    const int part = rank * WARPS + warp, parts = p.cluster * WARPS;
    const int rt0 = (int) ((long long) p.w.row_tiles * part / parts), rt1 = (int) ((long long) p.w.row_tiles * (part + 1) / parts);
    const T* dy = (const T*) p.in;

    // what a warp holds of one block row: a block's codes and, for its one or two groups, zero points of rows a and a + 8 and
    // scales of rows 2 t, 2 t + 8 and 2 t + 1, 2 t + 9
    constexpr int MINE = GROUPS == 4 ? 2 : 1;
    struct Row {
        uint32_t zeros[MINE], scales[MINE][2];
    };
    const int first = (kb & 1) * GROUPS / 2;  // the block's first group in its step
    auto load = [&](int rt, Row& r) {
        const long long at = ((long long) rt * p.w.steps + (kb >> 1)) * (16 * GROUPS);
#pragma unroll
        for (int m = 0; m < MINE; m++) {
            r.zeros[m] = p.w.zeros ? __ldg(reinterpret_cast<const uint16_t*>(p.w.zeros + at + (a * GROUPS + first + m) * 2)) : 0x0808u;
            r.scales[m][0] = __ldg(reinterpret_cast<const uint32_t*>(p.w.scales + at + (2 * t * GROUPS + first + m) * 2));
            r.scales[m][1] = __ldg(reinterpret_cast<const uint32_t*>(p.w.scales + at + ((2 * t + 1) * GROUPS + first + m) * 2));
        }
    };
    float total[4][NT][4] = {};
    const uint4* codes = p.w.codes + ((long long) rt0 * p.w.steps * 2 + kb) * 32 + lane;
    const long long stride = (long long) p.w.steps * 64;
#pragma unroll
    for (int i = 0; i < DX_AHEAD - 1; i++) {
        if (rt0 + i < rt1) fetch16(queue + i * 32, codes);
        codes += stride;
        fetch_commit();
    }
    Row next = {};
    if (rt0 < rt1) load(rt0, next);
    int slot = 0, free = DX_AHEAD - 1;
    for (int rt = rt0; rt < rt1; rt++) {
        const Row now = next;
        if (rt + DX_AHEAD - 1 < rt1) fetch16(queue + free * 32, codes);
        codes += stride;
        fetch_commit();
        if (rt + 1 < rt1) load(rt + 1, next);
        fetch_wait<DX_AHEAD - 1>();
        const uint4 c = queue[slot * 32];
        free = slot;
        slot = (slot + 1) % DX_AHEAD;
        const uint32_t words[4] = {c.x, c.y, c.z, c.w};
        // this lane's four output features: 16 rt + {2 t, 2 t + 1, 2 t + 8, 2 t + 9}
        float v[NT][4];
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            const int row = row0 + nt * 8 + a;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int n = rt * 16 + 2 * t + (i & 1) + (i >> 1) * 8;
                v[nt][i] = (row < p.rows && n < p.w.N) ? to_float(dy[row * p.ld_in + n]) : 0.f;
            }
        }
#pragma unroll
        for (int m = 0; m < MINE; m++) {
            const uint32_t s0 = now.scales[m][0], s1 = now.scales[m][1];
            const float s[4] = {q4_scale((uint16_t) s0, p.w.scale_bf16), q4_scale((uint16_t) s1, p.w.scale_bf16),
                                q4_scale((uint16_t) (s0 >> 16), p.w.scale_bf16), q4_scale((uint16_t) (s1 >> 16), p.w.scale_bf16)};
            uint32_t b[NT][2][TERMS];
#pragma unroll
            for (int nt = 0; nt < NT; nt++) {
                if constexpr (TERMS == 2) {
                    round_pair(v[nt][0] * s[0], v[nt][1] * s[1], b[nt][0]);
                    round_pair(v[nt][2] * s[2], v[nt][3] * s[3], b[nt][1]);
                } else {
                    split_pair<TERMS>(v[nt][0] * s[0], v[nt][1] * s[1], b[nt][0]);
                    split_pair<TERMS>(v[nt][2] * s[2], v[nt][3] * s[3], b[nt][1]);
                }
            }
            const uint32_t sub_lo = zero_pair<M>(now.zeros[m] & 15u), sub_hi = zero_pair<M>((now.zeros[m] >> 8) & 15u);
#pragma unroll
            for (int j = m * 4 / MINE; j < (m + 1) * 4 / MINE; j++) {
                uint32_t w[4], wt[4];
                unpack_centred<M>(words[j], sub_lo, sub_hi, w);
                // registers 0, 1 hold the lower pairs of rows 0-7, 8-15, registers 2, 3 the upper pairs; transposed, the
                // features are the rows of the A operand and 1 and 2 change places
                wt[0] = transpose8(w[0]); wt[1] = transpose8(w[2]); wt[2] = transpose8(w[1]); wt[3] = transpose8(w[3]);
#pragma unroll
                for (int nt = 0; nt < NT; nt++) {
                    float acc[4] = {};
#pragma unroll
                    for (int u = TERMS - 1; u >= 0; u--) mma<M>(acc, wt, b[nt][0][u], b[nt][1][u]);
#pragma unroll
                    for (int i = 0; i < 4; i++) total[j][nt][i] += acc[i];
                }
            }
        }
    }
    __syncthreads();  // all queues are empty
#pragma unroll
    for (int j = 0; j < 4; j++)
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int i = 0; i < 4; i++) red[warp * E + ((j * NT + nt) * 4 + i) * 32 + lane] = total[j][nt][i];
    __syncthreads();
#pragma unroll
    for (int e = threadIdx.x; e < E; e += WARPS * 32) {  // over the warps first
        float v = red[e];
#pragma unroll
        for (int w = 1; w < WARPS; w++) v += red[w * E + e];
        red[e] = v;
    }
    T* out = (T*) p.out;
    cluster_arrive();
    cluster_wait();
    join<E, 1, WARPS>(red, rank, p.cluster, [&](int e, float val) {
        const int l = e & 31, i = (e >> 5) & 3, nt = (e >> 7) % NT, j = (e >> 7) / NT;
        // row a of the transposed matrix is the feature of lane group a / 2, element a & 1 of its pair; rows 8..15 are the upper pairs
        const int ar = l >> 2;
        const int k = kb * 64 + 32 * (j >> 1) + 8 * (ar >> 1) + 4 * (j & 1) + 2 * (i >> 1) + (ar & 1);
        const int row = row0 + nt * 8 + (l & 3) * 2 + (i & 1);
        if (k >= p.w.K || row >= p.rows) return;
        out[row * p.ld_out + k] = from_float<T>(val);
    });
    cluster_arrive();  // nobody leaves while its sums may still be read
    cluster_wait();
}

// ------------------------------------------------------------------ quantising, packing, unpacking

// One warp per group of one row.  Symmetric: s = max|w| / 7, q = round(w / s) + 8.  With zero points: the range [min(w, 0),
// max(w, 0)] is cut into 15 steps, z = round(-low / s), q = round(w / s) + z.  The scale is rounded to its 16-bit type first
// and codes are taken with the rounded scale, so a code is the nearest one to the weight that the stored numbers allow.
template <typename T>
__global__ void __launch_bounds__(256)
q4_quantize_kernel(const T* __restrict__ W, long long ldw, int N, int K, int group, int groups, int scale_bf16, uint8_t* __restrict__ codes,
                   long long ldq, uint16_t* __restrict__ scales, uint8_t* __restrict__ zeros) {
    const long long item = ((long long) blockIdx.x * blockDim.x + threadIdx.x) >> 5;
    const int lane = threadIdx.x & 31;
    if (item >= (long long) N * groups) return;
    const int n = (int) (item / groups), g = (int) (item % groups);
    const int k0 = g * group, k1 = min(K, k0 + group);
    const T* row = W + n * ldw;
    float low = 0.f, high = 0.f;
    bool odd = false;  // a weight that is not finite makes the group's scale NaN
    for (int k = k0 + lane; k < k1; k += 32) {
        const float v = to_float(row[k]);
        odd |= !isfinite(v);
        low = fminf(low, v);
        high = fmaxf(high, v);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        low = fminf(low, __shfl_xor_sync(0xffffffffu, low, o));
        high = fmaxf(high, __shfl_xor_sync(0xffffffffu, high, o));
    }
    odd = __any_sync(0xffffffffu, odd);
    float s = zeros ? __fdiv_rn(high, 15.f) - __fdiv_rn(low, 15.f) : __fdiv_rn(fmaxf(high, -low), 7.f);
    uint16_t bits;
    if (scale_bf16) {
        bits = __bfloat16_as_ushort(__float2bfloat16_rn(s));
    } else {
        bits = __half_as_ushort(__float2half_rn(fminf(s, 65504.f)));
        if (bits == 0 && s > 0.f) bits = 1;  // the smallest scale there is, not zero
    }
    if (odd) bits = 0x7fffu;  // NaN in both types
    s = q4_scale(bits, scale_bf16);
    const float zf = zeros && s > 0.f ? fminf(fmaxf(rintf(__fdiv_rn(-low, s)), 0.f), 15.f) : (zeros ? 0.f : 8.f);
    const int z = (int) zf;
    if (lane == 0) {
        scales[(long long) n * groups + g] = bits;
        if (zeros) zeros[(long long) n * groups + g] = (uint8_t) z;
    }
    for (int k = k0 + 2 * lane; k < k1; k += 64) {
        uint32_t two = 0;
#pragma unroll
        for (int i = 0; i < 2; i++) {
            int q = z;
            if (k + i < k1 && s > 0.f) {
                const float v = rintf(__fdiv_rn(to_float(row[k + i]), s)) + zf;
                q = (int) fminf(fmaxf(v, 0.f), 15.f);
            }
            two |= (uint32_t) q << (4 * i);
        }
        codes[n * ldq + k / 2] = (uint8_t) two;  // groups start at even features: a byte belongs to one group
    }
}

// One thread per lane of a block: 32 codes gathered from two rows.
__global__ void __launch_bounds__(256)
q4_pack_kernel(const uint8_t* __restrict__ codes, long long ldq, int N, int K, int row_tiles, int blocks, uint4* __restrict__ out) {
    const long long i = (long long) blockIdx.x * blockDim.x + threadIdx.x;
    if (i >= (long long) row_tiles * blocks * 32) return;
    const int lane = (int) (i & 31), a = lane >> 2, t = lane & 3;
    const long long block = i >> 5;
    const int kb = (int) (block % blocks), rt = (int) (block / blocks);
    uint32_t words[4];
#pragma unroll
    for (int j = 0; j < 4; j++) {
        uint32_t w = 0;
#pragma unroll
        for (int f = 0; f < 4; f++) {
            const int n = rt * 16 + a + (f & 1) * 8;
            const int k = kb * 64 + 32 * (j >> 1) + 8 * t + 4 * (j & 1) + 2 * (f >> 1);
            uint32_t two = 0;
            if (n < N && k < K) two = codes[n * ldq + k / 2];
            if (k + 1 >= K) two &= 15u;
            w |= (two & 15u) << (4 * f) | (two >> 4) << (16 + 4 * f);
        }
        words[j] = w;
    }
    out[i] = make_uint4(words[0], words[1], words[2], words[3]);
}

__global__ void __launch_bounds__(256)
q4_pack_scales_kernel(const uint16_t* __restrict__ scales, const uint8_t* __restrict__ zeros, int groups_in, const Q4View w, uint16_t* __restrict__ out_s,
                      uint8_t* __restrict__ out_z) {
    const int per_step = 1 << (7 - w.group_shift);  // groups
    const long long i = (long long) blockIdx.x * blockDim.x + threadIdx.x;
    if (i >= (long long) w.row_tiles * w.steps * per_step * 16) return;
    const int local = (int) (i & 15);
    const long long at = i >> 4;
    const int g = (int) (at % ((long long) w.steps * per_step)), rt = (int) (at / ((long long) w.steps * per_step)), n = rt * 16 + local;
    const bool in = n < w.N && g < groups_in;
    const long long place = q4_scale_at(w, rt, g / per_step) + q4_scale_place(local, (g % per_step) << w.group_shift, w.group_shift);
    out_s[place] = in ? scales[(long long) n * groups_in + g] : 0;
    if (out_z) out_z[place] = in ? zeros[(long long) n * groups_in + g] : 0;
}

// One thread per lane of a block writes the 32 weights it holds.
template <typename T>
__global__ void __launch_bounds__(256)
q4_unpack_kernel(const Q4View w, T* __restrict__ out, long long ldo) {
    const long long i = (long long) blockIdx.x * blockDim.x + threadIdx.x;
    const int blocks = 2 * w.steps;
    if (i >= (long long) w.row_tiles * blocks * 32) return;
    const int lane = (int) (i & 31), a = lane >> 2, t = lane & 3;
    const long long block = i >> 5;
    const int kb = (int) (block % blocks), rt = (int) (block / blocks);
    const uint4 v = w.codes[i];
    const uint32_t words[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const long long at = q4_scale_at(w, rt, kb >> 1) + q4_scale_place(a, (kb & 1) * 64 + j * 16, w.group_shift);
#pragma unroll
        for (int f = 0; f < 4; f++) {
            const int n = rt * 16 + a + (f & 1) * 8;
            const int k = kb * 64 + 32 * (j >> 1) + 8 * t + 4 * (j & 1) + 2 * (f >> 1);
            const float s = q4_scale(w.scales[at + (f & 1)], w.scale_bf16);
            const int z = w.zeros ? (w.zeros[at + (f & 1)] & 15) : 8;
            if (n < w.N && k < w.K) out[n * ldo + k] = from_float<T>(s * (float) ((int) (words[j] >> (4 * f) & 15u) - z));
            if (n < w.N && k + 1 < w.K) out[n * ldo + k + 1] = from_float<T>(s * (float) ((int) (words[j] >> (16 + 4 * f) & 15u) - z));
        }
    }
}

// ------------------------------------------------------------------ host side

int bad(const char* who, const char* what) {
    set_error("%s: %s", who, what);
    return CAKEB200_ERR_ARG;
}

bool known_type(int type) { return type == CAKEB200_F32 || type == CAKEB200_F16 || type == CAKEB200_BF16; }

int check_geometry(const char* who, int N, int K, int group, int scale_type) {
    if (N <= 0 || K <= 0) return bad(who, "features must be positive");
    if (group != 32 && group != 64 && group != 128) return bad(who, "the group is 32, 64 or 128 input features");
    if (scale_type != CAKEB200_F16 && scale_type != CAKEB200_BF16) return bad(who, "scales are float16 or bfloat16");
    if (K > (1 << 30) || N > (1 << 30)) {
        set_error("%s: more than 2^30 features", who);
        return CAKEB200_ERR_TOO_LARGE;
    }
    return CAKEB200_OK;
}

size_t codes_bytes(int N, int K) { return (size_t) q4_row_tiles(N) * q4_steps(K) * 1024; }
size_t scales_count(int N, int K, int group) { return (size_t) q4_row_tiles(N) * q4_steps(K) * (128 / group) * 16; }
int shift_of(int group) { return group == 32 ? 5 : group == 64 ? 6 : 7; }

int blocks_for(const char* who, long long threads, unsigned* out) {
    const long long b = (threads + 255) / 256;
    if (b > 0x7fffffffLL) {
        set_error("%s: the matrix is too large for one launch", who);
        return CAKEB200_ERR_TOO_LARGE;
    }
    *out = (unsigned) b;
    return CAKEB200_OK;
}

template <typename K>
int launch_clustered(K kernel, unsigned x, unsigned y, int cluster, int warps, size_t smem, const Q4Args& args, cudaStream_t s) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(x, y);
    cfg.blockDim = dim3((unsigned) warps * 32);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned) cluster;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    CAKE_CUDA_OK(cudaLaunchKernelEx(&cfg, kernel, args));
    return CAKEB200_OK;
}
// CTAs of a cluster that share out the reduction: at least `least`, and more while there are fewer than `wanted` CTAs and each
// of the cluster's warps still has `per_warp` steps (block rows) of it.
int pick_cluster(long long items, int depth, int warps, int per_warp, int least, long long wanted) {
    int c = 1;
    while (c < MAX_CLUSTER && depth >= 2 * c * warps * per_warp && (c < least || items * c < wanted)) c *= 2;
    return c;
}

// The forward product runs CTAs of four warps, as many as fit, two or more to a cluster.  Times in us over warps per CTA x CTAs per
// cluster x CTAs per SM, one row: 16384 x 16384 FP32 4x1x4 90, 4x2x4 79, 8x1x2 89, 8x2x2 77, 8x4x2 133; 16384 x 8192 BF16
// 4x1x4 33, 4x2x4 30, 4x2x5 27, 8x1x2 33, 8x2x2 30; 4096 x 4096 FP16 4x1 9.1, 4x2 7.2, 4x4 6.5; 2048 x 2048 BF16 4x1 6.4,
// 4x2 4.8, 4x4 4.7.
constexpr int LINEAR_WARPS = 4;

// One wave: as many clusters as the device holds of this kernel (asked once per device and cluster size), or one per item.
template <typename T, int NT, int R, int GROUPS>
int launch_linear_as(Q4Args& p, long long items, int device, cudaStream_t s) {
    static std::atomic<int> known[64][4];  // by device and log2 of the cluster size
    const auto kernel = q4_linear_kernel<T, NT, R, GROUPS, LINEAR_WARPS>;
    constexpr size_t smem = (size_t) LINEAR_WARPS * (AHEAD * R * 1024 + 2 * R * NT * 512);
    const int log2 = p.cluster == 1 ? 0 : p.cluster == 2 ? 1 : p.cluster == 4 ? 2 : 3;
    int fit = device < 64 ? known[device][log2].load() : 0;
    if (fit == 0) {
        CAKE_CUDA_OK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int) smem));
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3((unsigned) p.cluster);
        cfg.blockDim = dim3(LINEAR_WARPS * 32);
        cfg.dynamicSmemBytes = smem;
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = (unsigned) p.cluster;
        attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        CAKE_CUDA_OK(cudaOccupancyMaxActiveClusters(&fit, kernel, &cfg));
        if (fit < 1) {
            set_error("q4_linear: the kernel does not fit the device");
            return CAKEB200_ERR_CUDA;
        }
        if (device < 64) known[device][log2] = fit;
    }
    const unsigned grid = (unsigned) (std::min<long long>(items, fit) * p.cluster);
    return launch_clustered(kernel, grid, 1, p.cluster, LINEAR_WARPS, smem, p, s);
}
template <typename T, int NT>
int launch_linear_rows(Q4Args& p, const DeviceState* st, cudaStream_t s) {
    constexpr int R = 2;
    p.chunks = (p.rows + 8 * NT - 1) / (8 * NT);
    const long long items = (long long) (p.w.row_tiles / R) * p.chunks;
    p.cluster = pick_cluster(items, p.w.steps, LINEAR_WARPS, 1, 2, 2LL * st->sm_count);
    if (p.w.group_shift == 7) return launch_linear_as<T, NT, R, 1>(p, items, st->device, s);
    if (p.w.group_shift == 6) return launch_linear_as<T, NT, R, 2>(p, items, st->device, s);
    return launch_linear_as<T, NT, R, 4>(p, items, st->device, s);
}
template <typename T>
int launch_linear(Q4Args& p, const DeviceState* st, cudaStream_t s) {
    if (p.rows <= 8) return launch_linear_rows<T, 1>(p, st, s);
    if (p.rows <= 16) return launch_linear_rows<T, 2>(p, st, s);
    return launch_linear_rows<T, 4>(p, st, s);
}

// The gradient's CTAs have eight warps and one block of 64 input features each.  us over warps per CTA x CTAs per cluster, one row:
// 16384 x 8192 BF16 4x1 183, 4x4 58, 8x1 100, 8x4 52, 8x8 52; 4096 x 4096 FP32 4x1 34, 8x4 10.1, 8x8 10.5; 2048 x 2048 FP32
// 8x1 11.3, 8x4 5.6, 8x8 5.0.
constexpr int DX_WARPS = 8;
template <typename T, int NT>
int launch_dx_rows(Q4Args& p, int sm_count, cudaStream_t s) {
    const unsigned blocks = 2u * (unsigned) p.w.steps, chunks = (unsigned) ((p.rows + 8 * NT - 1) / (8 * NT));
    p.cluster = pick_cluster((long long) blocks * chunks, p.w.row_tiles, DX_WARPS, 1, 1, 4LL * sm_count);
    const unsigned x = blocks * (unsigned) p.cluster;
    if (p.w.group_shift == 7) return launch_clustered(q4_linear_dx_kernel<T, NT, 1, DX_WARPS>, x, chunks, p.cluster, DX_WARPS, 0, p, s);
    if (p.w.group_shift == 6) return launch_clustered(q4_linear_dx_kernel<T, NT, 2, DX_WARPS>, x, chunks, p.cluster, DX_WARPS, 0, p, s);
    return launch_clustered(q4_linear_dx_kernel<T, NT, 4, DX_WARPS>, x, chunks, p.cluster, DX_WARPS, 0, p, s);
}
template <typename T>
int launch_dx(Q4Args& p, int sm_count, cudaStream_t s) {
    return p.rows <= 8 ? launch_dx_rows<T, 1>(p, sm_count, s) : launch_dx_rows<T, 2>(p, sm_count, s);
}

// Common checks of the two products.  in_cols / out_cols: row lengths of the operand and of the result.
int product(const char* who, const cakeb200_q4* w, const void* in, long long ld_in, const void* bias, void* out, long long ld_out,
            int rows, int type, bool dx, void* workspace, size_t workspace_bytes, void* stream) {
    *thread_stats() = cakeb200_stats();
    Q4Args p = {};
    int rc = q4_view(w, who, &p.w);
    if (rc) return rc;
    if (!known_type(type)) return bad(who, "the type is float32, float16 or bfloat16");
    if (rows < 0) return bad(who, "negative number of rows");
    if (rows == 0) return CAKEB200_OK;
    if (!in || !out) return bad(who, "null pointer");
    const int in_cols = dx ? p.w.N : p.w.K, out_cols = dx ? p.w.K : p.w.N;
    if (rows > 1 && (ld_in < in_cols || ld_out < out_cols)) return bad(who, "a leading dimension is smaller than its row");
    DeviceState* st = device_state();
    if (!st) return CAKEB200_ERR_NO_DEVICE;
    if (!on_current_device(w->packed) || !on_current_device(in) || !on_current_device(out) || (bias && !on_current_device(bias)))
        return bad(who, "operands must be device pointers of the current device");
    const size_t size = type == CAKEB200_F32 ? 4 : 2;
    if ((uintptr_t) in % size || (uintptr_t) out % size || (uintptr_t) bias % size) return bad(who, "a pointer is not aligned to its type");
    p.in = in; p.out = out; p.bias = bias;
    p.ld_in = ld_in; p.ld_out = ld_out; p.rows = rows;
    p.vec = (uintptr_t) in % 16 == 0 && (rows == 1 || (ld_in * (long long) size) % 16 == 0);
    cudaStream_t s = (cudaStream_t) stream;
    if (!few_rows(p.w, rows, type, dx)) {
        if (!workspace || (uintptr_t) workspace % 1024) return bad(who, "this many rows need a workspace on a 1024-byte boundary");
        if (workspace_bytes < q4_gemm_workspace(p.w, rows, type, dx)) return bad(who, "the workspace is too small");
        if (!on_current_device(workspace)) return bad(who, "operands must be device pointers of the current device");
        return launch_q4_gemm(p.w, in, ld_in, bias, out, ld_out, rows, type, dx, workspace, st, s);
    }
    if (dx)
        rc = type == CAKEB200_F32 ? launch_dx<float>(p, st->sm_count, s)
             : type == CAKEB200_F16 ? launch_dx<__half>(p, st->sm_count, s) : launch_dx<__nv_bfloat16>(p, st->sm_count, s);
    else
        rc = type == CAKEB200_F32 ? launch_linear<float>(p, st, s)
             : type == CAKEB200_F16 ? launch_linear<__half>(p, st, s) : launch_linear<__nv_bfloat16>(p, st, s);
    if (!rc) thread_stats()->launches = 1;
    return rc;
}

}  // namespace

bool on_current_device(const void* p) {
    int dev = -1;
    cudaPointerAttributes a;
    if (cudaGetDevice(&dev) != cudaSuccess || cudaPointerGetAttributes(&a, p) != cudaSuccess) {
        cudaGetLastError();
        return false;
    }
    return a.type == cudaMemoryTypeManaged || (a.type == cudaMemoryTypeDevice && a.device == dev);
}

int q4_view(const cakeb200_q4* w, const char* who, Q4View* out) {
    if (!w || !w->packed) return bad(who, "null weights");
    int rc = check_geometry(who, w->out_features, w->in_features, w->group, w->scale_type);
    if (rc) return rc;
    if ((uintptr_t) w->packed % 16) return bad(who, "packed weights start on a 16-byte boundary");
    out->N = w->out_features;
    out->K = w->in_features;
    out->group_shift = shift_of(w->group);
    out->row_tiles = q4_row_tiles(out->N);
    out->steps = q4_steps(out->K);
    out->scale_bf16 = w->scale_type == CAKEB200_BF16;
    const char* base = (const char*) w->packed;
    out->codes = (const uint4*) base;
    out->scales = (const uint16_t*) (base + codes_bytes(out->N, out->K));
    out->zeros = w->has_zeros ? (const uint8_t*) (out->scales + scales_count(out->N, out->K, w->group)) : nullptr;
    return CAKEB200_OK;
}

}  // namespace cakeb200

using namespace cakeb200;

extern "C" {

size_t cakeb200_q4_packed_bytes(int out_features, int in_features, int group, int has_zeros) {
    if (check_geometry("cakeb200_q4_packed_bytes", out_features, in_features, group, CAKEB200_F16)) return 0;
    return codes_bytes(out_features, in_features) + scales_count(out_features, in_features, group) * (has_zeros ? 3 : 2);
}

int cakeb200_q4_quantize(const void* W, long long ldw, int type, int out_features, int in_features, int group, int scale_type,
                         void* codes, long long ldq, void* scales, void* zeros, void* stream) {
    static const char* who = "cakeb200_q4_quantize";
    *thread_stats() = cakeb200_stats();
    int rc = check_geometry(who, out_features, in_features, group, scale_type);
    if (rc) return rc;
    if (!W || !codes || !scales) return bad(who, "null pointer");
    if (!known_type(type)) return bad(who, "the type is float32, float16 or bfloat16");
    if (ldw < in_features || ldq < (in_features + 1) / 2) return bad(who, "a leading dimension is smaller than its row");
    DeviceState* st = device_state();
    if (!st) return CAKEB200_ERR_NO_DEVICE;
    if (!on_current_device(W) || !on_current_device(codes) || !on_current_device(scales) || (zeros && !on_current_device(zeros)))
        return bad(who, "operands must be device pointers of the current device");
    const int groups = (in_features + group - 1) / group;
    unsigned blocks;
    if ((rc = blocks_for(who, (long long) out_features * groups * 32, &blocks))) return rc;
    cudaStream_t s = (cudaStream_t) stream;
    const int bf = scale_type == CAKEB200_BF16;
    if (type == CAKEB200_F32)
        q4_quantize_kernel<float><<<blocks, 256, 0, s>>>((const float*) W, ldw, out_features, in_features, group, groups, bf, (uint8_t*) codes, ldq,
                                                         (uint16_t*) scales, (uint8_t*) zeros);
    else if (type == CAKEB200_F16)
        q4_quantize_kernel<__half><<<blocks, 256, 0, s>>>((const __half*) W, ldw, out_features, in_features, group, groups, bf, (uint8_t*) codes, ldq,
                                                          (uint16_t*) scales, (uint8_t*) zeros);
    else
        q4_quantize_kernel<__nv_bfloat16><<<blocks, 256, 0, s>>>((const __nv_bfloat16*) W, ldw, out_features, in_features, group, groups, bf,
                                                                 (uint8_t*) codes, ldq, (uint16_t*) scales, (uint8_t*) zeros);
    CAKE_CUDA_OK(cudaGetLastError());
    thread_stats()->launches = 1;
    return CAKEB200_OK;
}

int cakeb200_q4_pack(const void* codes, long long ldq, const void* scales, const void* zeros, int out_features, int in_features, int group,
                     int scale_type, void* packed, void* stream) {
    static const char* who = "cakeb200_q4_pack";
    *thread_stats() = cakeb200_stats();
    int rc = check_geometry(who, out_features, in_features, group, scale_type);
    if (rc) return rc;
    if (!codes || !scales || !packed) return bad(who, "null pointer");
    if (ldq < (in_features + 1) / 2) return bad(who, "a leading dimension is smaller than its row");
    if ((uintptr_t) packed % 16) return bad(who, "packed weights start on a 16-byte boundary");
    DeviceState* st = device_state();
    if (!st) return CAKEB200_ERR_NO_DEVICE;
    if (!on_current_device(codes) || !on_current_device(scales) || !on_current_device(packed) || (zeros && !on_current_device(zeros)))
        return bad(who, "operands must be device pointers of the current device");
    const cakeb200_q4 desc = {packed, out_features, in_features, group, scale_type, zeros != nullptr};
    Q4View v;
    if ((rc = q4_view(&desc, who, &v))) return rc;
    unsigned b0, b1;
    if ((rc = blocks_for(who, (long long) v.row_tiles * v.steps * 64, &b0)) ||
        (rc = blocks_for(who, (long long) scales_count(out_features, in_features, group), &b1)))
        return rc;
    cudaStream_t s = (cudaStream_t) stream;
    q4_pack_kernel<<<b0, 256, 0, s>>>((const uint8_t*) codes, ldq, out_features, in_features, v.row_tiles, 2 * v.steps, (uint4*) packed);
    CAKE_CUDA_OK(cudaGetLastError());
    q4_pack_scales_kernel<<<b1, 256, 0, s>>>((const uint16_t*) scales, (const uint8_t*) zeros, (in_features + group - 1) / group, v,
                                             (uint16_t*) v.scales, (uint8_t*) v.zeros);
    CAKE_CUDA_OK(cudaGetLastError());
    thread_stats()->launches = 2;
    return CAKEB200_OK;
}

int cakeb200_q4_dequantize(const cakeb200_q4* w, void* W, long long ldw, int type, void* stream) {
    static const char* who = "cakeb200_q4_dequantize";
    *thread_stats() = cakeb200_stats();
    Q4View v;
    int rc = q4_view(w, who, &v);
    if (rc) return rc;
    if (!W) return bad(who, "null pointer");
    if (!known_type(type)) return bad(who, "the type is float32, float16 or bfloat16");
    if (ldw < v.K) return bad(who, "a leading dimension is smaller than its row");
    DeviceState* st = device_state();
    if (!st) return CAKEB200_ERR_NO_DEVICE;
    if (!on_current_device(w->packed) || !on_current_device(W)) return bad(who, "operands must be device pointers of the current device");
    unsigned blocks;
    if ((rc = blocks_for(who, (long long) v.row_tiles * v.steps * 64, &blocks))) return rc;
    cudaStream_t s = (cudaStream_t) stream;
    if (type == CAKEB200_F32) q4_unpack_kernel<float><<<blocks, 256, 0, s>>>(v, (float*) W, ldw);
    else if (type == CAKEB200_F16) q4_unpack_kernel<__half><<<blocks, 256, 0, s>>>(v, (__half*) W, ldw);
    else q4_unpack_kernel<__nv_bfloat16><<<blocks, 256, 0, s>>>(v, (__nv_bfloat16*) W, ldw);
    CAKE_CUDA_OK(cudaGetLastError());
    thread_stats()->launches = 1;
    return CAKEB200_OK;
}

size_t cakeb200_q4_workspace(const cakeb200_q4* w, int rows, int type, int dx) {
    Q4View v;
    if (q4_view(w, "cakeb200_q4_workspace", &v) || !known_type(type) || few_rows(v, rows, type, dx != 0)) return 0;
    return q4_gemm_workspace(v, rows, type, dx != 0);
}

int cakeb200_q4_linear(const cakeb200_q4* w, const void* x, long long ldx, const void* bias, void* y, long long ldy, int rows, int type,
                       void* workspace, size_t workspace_bytes, void* stream) {
    return product("cakeb200_q4_linear", w, x, ldx, bias, y, ldy, rows, type, false, workspace, workspace_bytes, stream);
}

int cakeb200_q4_linear_dx(const cakeb200_q4* w, const void* dy, long long lddy, void* dx, long long lddx, int rows, int type, void* workspace,
                          size_t workspace_bytes, void* stream) {
    return product("cakeb200_q4_linear_dx", w, dy, lddy, nullptr, dx, lddx, rows, type, true, workspace, workspace_bytes, stream);
}

}  // extern "C"
