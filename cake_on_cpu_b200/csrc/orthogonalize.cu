// Orthogonalising an update by Newton-Schulz products, alone and inside an optimiser's step.
//
//     X_0 = G / (|G|_F + eps);    P = X X^T;    Q = a I + b P + c P P;    X <- Q X;    `steps` times.
//
// Every singular value s of X goes to a s + b s^3 + c s^5, the singular vectors stay: with the usual coefficients values
// anywhere in (0, 1] end up around 1.  X is taken m x n with m <= n (the transpose of a tall G), so that P is the smaller
// square.  P and Q are symmetric: only the tiles on and below the diagonal are computed, 2 m^2 n + m^3 multiply-adds
// per step instead of 2 m^2 n + 2 m^3 and an elementwise pass.  The polynomial lives in the second product's epilogue, which
// adds b P and a I to c P P in FP32.
//
// All matrices between the first and the last kernel are pairs of FP16 planes (plane_gemm.cuh), 22 bits and a sign: three
// MMAs per product.  Small singular values grow by a factor a = 3.4 per step, 480 in five, and so does the rounding noise
// of X beside them: a single 16-bit plane (2^-9 or 2^-12) would leave per cents of noise in the result, pairs leave what FP32
// products leave.  The range of FP16 is no limit: X, P and Q are held with powers of two taken out (Exponents below) that follow from
// bounds of the singular values, so that none overflows and a small X, as of a G far below eps, keeps its bits.  Nothing is ever
// transposed or mirrored in memory: Q X reads X, and the upper triangles of P and Q are read, down the columns of what is there
// (an SM stores 32 bytes a clock, so bytes written are what an epilogue costs).
#include <cmath>

#include "plane_gemm.cuh"

namespace cakeb200 {

using plane::Planes;
using plane::TileAt;

namespace {

using plane::Fp16Planes;

constexpr int TERMS = 2;
constexpr int NORM_BLOCKS = 512;  // room for partial sums of squares per matrix; the last place is `SHIFT_AT`
constexpr int SHIFT_AT = NORM_BLOCKS - 1;
constexpr int MAX_STEPS = 64;

// How the matrices are held: X as 2^(up - x) X, P as 2^(-2 x) P and Q as 2^-q Q, with x and q a step's exponents such that the singular values
// of X are below 2^x and those of Q below 2^q.  X_0 has singular values up to |G| / (|G| + eps) <= 1; the host follows the
// largest that the polynomial makes of (0, 1] (`x`, `q`).  A G below eps begins at 2^-shift, which only the device knows, and grows
// by 2^q a step until it meets the host's bound.  2^up, around sqrt(m n), puts the elements of X, not the singular values, around 1.
struct Exponents {
    short x[MAX_STEPS + 1], q[MAX_STEPS];
    short a, b, c;  // |a| < 2^a and so on; far below everything where the coefficient is zero
    short up;
};
constexpr int FAR_BELOW = -8000;
struct StepExponents {
    int x, q, next;  // x of the step and of the one after it
};
__device__ __forceinline__ void begin(const Exponents& e, int shift, StepExponents& s) { s.next = min((int) e.x[0], -shift); }
__device__ __forceinline__ void advance(const Exponents& e, int q, int next, StepExponents& s) {
    s.x = s.next;
    const int b = e.b + 2 * s.x, c = e.c + 4 * s.x;  // |a| + |b| 4^x + |c| 16^x
    const int bound = max((int) e.a, max(b, c)) + (e.a >= max(b, c) + 2 ? 1 : 2);
    s.q = min(q, bound);
    s.next = min(next, s.x + s.q);
}
__device__ __forceinline__ StepExponents exponents_of(const Exponents& e, int shift, int step) {
    StepExponents s;
    begin(e, shift, s);
    for (int i = 0; i <= step; i++) advance(e, e.q[i], e.x[i + 1], s);
    return s;
}
// k 2^e for e between -252 and 254; beyond, zero and infinity (but a coefficient of zero stays zero)
__device__ __forceinline__ float times_power(float k, int e) {
    auto power = [](int e) { return __int_as_float(e < -126 ? 0 : e > 127 ? 0x7f800000 : (e + 127) << 23); };
    return k == 0.f ? 0.f : k * power(e >> 1) * power(e - (e >> 1));
}
__device__ __forceinline__ double power_of_two(int e) { return __hiloint2double((e + 1023) << 20, 0); }
// The factor that makes 2^(up + shift) X_0 of a matrix of that norm: 2^-shift is the first power of two at or above norm / (norm + eps).
__device__ __forceinline__ double first_factor(double norm, double eps, int up, int& shift) {
    const double inverse = 1.0 / (norm + eps), r = norm * inverse;
    shift = r > 0 && r < 1 ? min(1022 - (__double2hiint(r) >> 20), 100) : 0;  // no finite norm, or none at all: 0
    return inverse * power_of_two(up + shift);
}

// K blocks of 64 between folds of the main accumulator, whatever the result's type: one, or two where X has more than 512 rows.
// Errors of FP32 with folds every 64 / 128 of K (and of a plain FP32 evaluation): 137 x 900 1.3e-6 / 2.3e-6 (1.5e-6), 300 x 400 0.9e-6 /
// 1.3e-6 (2.0e-6), 700 x 800 0.9e-6 / 1.3e-6 (2.5e-6), 4096 x 4096 1.1e-6 / 1.4e-6 (4.8e-6); times 300 x 400 206 / 201 us, 2048 x 2048
// 624 / 580, 4096 x 4096 3.39 / 3.12 ms.
inline int fold_for(int m) { return m > 512 ? 2 : 1; }
// The tensor core truncates the sum that it adds to, which has a sign where sums do not: it is put back into the two products whose
// sums are of squares, by the additions that they really had, as measured in 2^-24 of the sum.
//   X X^T: sums that grow evenly lose 2.2, 3.0, 3.9 and 7.9 in 2, 3, 4 and 8 additions (rows of 32 to 256 random values).
//   P P: the largest product of a sum on the diagonal is there from some addition on, and all later ones take from the whole: 1.8 for
//   each but one in folds of 64 (5.5 in four, from the bias of single steps), 1.2 in folds of 128 (errors of 2048 x 2048 1.25e-6,
//   with 1.8 1.5e-6).
// A sum of a single addition is left alone, and so is Q X, whose sums are of either sign and, while X is small, of a single term.
// Errors over those of a plain FP32 evaluation, gradients of 32 to 128 rows and up to 2048 columns: median 0.90, 90 % below 1.22; with
// 0.36 (n + 1) in both products instead 1.31 and 1.94.  Matrices with one entry a row have nothing to put back and pay for it: 2e-6.
__device__ __forceinline__ plane::Loss gram_loss() { return {0.96f * 5.9604645e-8f, 0}; }
__device__ __forceinline__ plane::Loss square_loss(int fold) { return {(fold > 1 ? 1.2f : 1.8f) * 5.9604645e-8f, 1}; }
__device__ __forceinline__ plane::Loss no_loss() { return {0.f, 0}; }

// eight consecutive elements; `vec`: all eight exist and the address is 16-byte aligned
__device__ __forceinline__ void get8(const float* p, int n, bool vec, float* v) {
    if (vec && n >= 8) {
        const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
        v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    } else {
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] = e < n ? p[e] : 0.f;
    }
}
__device__ __forceinline__ void get8(const __nv_bfloat16* p, int n, bool vec, float* v) {
    if (vec && n >= 8) {
        const uint4 a = *reinterpret_cast<const uint4*>(p);
        const uint32_t u[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
        for (int e = 0; e < 4; e++) {
            v[2 * e] = __uint_as_float(u[e] << 16);
            v[2 * e + 1] = __uint_as_float(u[e] & 0xffff0000u);
        }
    } else {
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] = e < n ? __bfloat162float(p[e]) : 0.f;
    }
}
__device__ __forceinline__ void put8(float* p, int n, bool vec, const float* v) {
    if (vec && n >= 8) {
        reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
        reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
    } else {
#pragma unroll
        for (int e = 0; e < 8; e++)
            if (e < n) p[e] = v[e];
    }
}
// ------------------------------------------------------------------ the input: norm, momentum, planes

// A matrix (or a batch) in the caller's memory; vec: rows start on 16-byte boundaries.
template <typename T>
struct Matrix {
    T* base;
    long long ld, stride;
    int vec;
};

// What is orthogonalised: G itself, or the update U made of G and the momentum M.
template <typename T>
struct Source {
    Matrix<const T> g;
    float* m;          // nullptr: plain G
    long long ldm;
    int vec_m;
    float mu, rest;    // momentum and 1 - momentum, each rounded once
    int nesterov;
    int rows, cols;
};

// Eight values of row r from column c on.  UPDATE: M <- mu M + (1 - mu) G on the way (else M has it already).
template <typename T, bool UPDATE>
__device__ __forceinline__ void source8(const Source<T>& s, int batch, int r, int c, float* v) {
    const int n = s.cols - c;
    get8(s.g.base + batch * s.g.stride + r * s.g.ld + c, n, s.g.vec, v);
    if (s.m == nullptr) return;
    float m[8];
    float* at = s.m + r * s.ldm + c;
    get8(at, n, s.vec_m, m);
    if (UPDATE) {
#pragma unroll
        for (int e = 0; e < 8; e++) m[e] = s.mu * m[e] + s.rest * v[e];
        put8(at, n, s.vec_m, m);
    }
#pragma unroll
    for (int e = 0; e < 8; e++) v[e] = s.nesterov ? s.mu * m[e] + s.rest * v[e] : m[e];
}

// partial[batch][block] = sum of squares, in 64 bits: an FP32 sum of squares overflows and underflows long before G does.
template <typename T>
__global__ void __launch_bounds__(256)
norm_kernel(const Source<T> s, double* __restrict__ partial) {
    const int batch = blockIdx.y, segments = (s.cols + 7) / 8;
    const long long total = (long long) s.rows * segments;
    double sum = 0;
    for (long long i = (long long) blockIdx.x * 256 + threadIdx.x; i < total; i += (long long) gridDim.x * 256) {
        const int r = (int) (i / segments), c = (int) (i - (long long) r * segments) * 8;
        float v[8];
        source8<T, true>(s, batch, r, c, v);
#pragma unroll
        for (int e = 0; e < 8; e++)
            if (c + e < s.cols) sum += (double) v[e] * v[e];
    }
    __shared__ double warps[8];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if ((threadIdx.x & 31) == 0) warps[threadIdx.x >> 5] = sum;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < 8; w++) sum += warps[w];
        partial[batch * NORM_BLOCKS + blockIdx.x] = sum;
    }
}

// Planes of 2^(up + shift) X_0, which is the transpose of the source where that is `tall`; a warp does one 32 x 32 block.
template <typename T>
__global__ void __launch_bounds__(256)
split_kernel(const Source<T> s, double* partial, int partials, float eps, int up, bool tall, const Planes x, unsigned* arrived) {
    __shared__ float patches[8][plane::PATCH_FLOATS];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, batch = blockIdx.z;
    const int row0 = blockIdx.y * 32, col0 = (blockIdx.x * 8 + warp) * 32;
    if (col0 >= s.cols) return;
    plane::wait_for_previous_kernel();
    if (blockIdx.x == 0 && blockIdx.y == 0 && batch == 0 && threadIdx.x == 0) arrived[0] = arrived[1] = 0;  // for the barriers of the chain
    double sum = 0;
    for (int i = lane; i < partials; i += 32) sum += partial[batch * NORM_BLOCKS + i];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    int shift;
    const double inverse = first_factor(sqrt(sum), eps, up, shift);
    if (blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0) partial[batch * NORM_BLOCKS + SHIFT_AT] = shift;
    float* patch = patches[warp];
#pragma unroll
    for (int q = 0; q < 4; q++) {
        const int rl = 8 * q + (lane >> 2), cl = 8 * (lane & 3), r = row0 + rl, c = col0 + cl;
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] = 0.f;
        if (r < s.rows && c < s.cols) {
            source8<T, false>(s, batch, r, c, v);
#pragma unroll
            for (int e = 0; e < 8; e++) v[e] = (float) ((double) v[e] * inverse);
            if (!tall) plane::store8<Fp16Planes, TERMS>(x, batch, r, c, v);
        }
        if (tall) {
#pragma unroll
            for (int e = 0; e < 8; e++) patch[rl * plane::PATCH_LD + cl + e] = v[e];
        }
    }
    if (!tall) return;
    __syncwarp();
#pragma unroll
    for (int q = 0; q < 4; q++) {
        const int r = col0 + 8 * q + (lane >> 2), c = row0 + 8 * (lane & 3);
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] = patch[(8 * (lane & 3) + e) * plane::PATCH_LD + 8 * q + (lane >> 2)];
        if (r < s.cols && c < s.rows) plane::store8<Fp16Planes, TERMS>(x, batch, r, c, v);
    }
}

// ------------------------------------------------------------------ what becomes of the last X

__device__ __forceinline__ float get(const float* p) { return *p; }
__device__ __forceinline__ float get(const __nv_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ void put(float* p, float v) { *p = v; }
__device__ __forceinline__ void put(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

// the last X, f times the product, rounded once to the result's type
template <typename T>
struct ResultEpilogue {
    struct Args {
        Matrix<T> out;
        int rows, cols;
    };
    // one value of the block's row r, in the lane's column of it
    struct Writer {
        T* p;
        long long ld;
        int rows;
        float f;
        __device__ __forceinline__ void operator()(int r, float x) const {
            if (r < rows) put(p + r * ld, f * x);
        }
    };
    static __device__ __forceinline__ Writer writer(const Args& a, const TileAt& at, int lane, float f) {
        return {a.out.base + at.batch * a.out.stride + at.row * a.out.ld + at.col + lane, a.out.ld, at.col + lane < a.cols ? a.rows - at.row : 0, f};
    }
};

// W <- keep W - step X, the last X f times the product
template <typename T>
struct StepEpilogue {
    struct Args {
        Matrix<T> w;
        int rows, cols;
        float keep, step;
    };
    struct Writer {
        T* p;
        long long ld;
        int rows;
        float f, keep, step;
        __device__ __forceinline__ void operator()(int r, float x) const {
            if (r < rows) put(p + r * ld, keep * get(p + r * ld) - step * (f * x));
        }
    };
    static __device__ __forceinline__ Writer writer(const Args& a, const TileAt& at, int lane, float f) {
        return {a.w.base + at.row * a.w.ld + at.col + lane, a.w.ld, at.col + lane < a.cols ? a.rows - at.row : 0, f, a.keep, a.step};
    }
};

// ------------------------------------------------------------------ the chain of products

// One kernel runs all products of all steps (a launch each cost 4 us and more beside its 5 to 40 us of work, and ran its
// epilogue from a cold instruction cache).  CTAs meet at a grid-wide barrier between products: the drain warps of a CTA
// count it in when their stores are done, the TMA thread and the drain warps wait for the count.  The launch is
// cooperative, so that all CTAs are resident; waits are bounded.
//
enum { X_ROWS, X_COLUMNS, P_SYM, Q_SYM };  // what an operand is: X, its transpose, P, Q
struct Product : plane::Tiling {
    int a, b;
};

struct Chain {
    Planes x[2], p, q;           // step s reads x[s % 2] and writes the other
    Product gram, poly, apply, last;
    int batch, steps, fold;
    float ka, kb, kc;
    Exponents exponents;
    const double* shifts;        // per matrix, at SHIFT_AT of its NORM_BLOCKS
    float* parts;                // of cut tiles: [slot][32 x 32 block][1024]
    unsigned* arrived;           // CTAs that have come to the barriers so far; next to it, whether one came with work undone
    int mute;                    // self-test: the first CTA never multiplies
    int* status_word;
};

struct Maps {
    plane::OperandMaps x[2], p, q;
};

using plane::Item;
using plane::item_at;
using plane::place;

// Stores of this thread become visible to loads of other SMs, TMA among them, once the CTA has been counted in.
__device__ __forceinline__ void publish() { asm volatile("fence.proxy.async.global;\n\tfence.acq_rel.gpu;" ::: "memory"); }
__device__ __forceinline__ void count_in(unsigned* counter) { asm volatile("red.release.gpu.global.add.u32 [%0], 1;" ::"l"(counter) : "memory"); }
// Waits until `target` CTAs have been counted in (bounded, as the waits of plane_gemm.cuh).
__device__ __forceinline__ bool wait_for_count(const unsigned* counter, unsigned target, volatile int* abort_flag, int* status_word) {
    const unsigned long long t0 = ptx::global_ns();
    for (int spins = 1;; spins++) {
        unsigned v;
        asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(v) : "l"(counter) : "memory");
        if ((int) (v - target) >= 0) break;
        if ((spins & 255) == 0) {
            if (*abort_flag) return false;
            if ((long long) (ptx::global_ns() - t0) > ptx::WAIT_LIMIT_NS) {
                *abort_flag = 1;
                if (atomicCAS(status_word, 0, 1) == 0) {
                    status_word[1] = 550;
                    status_word[2] = (int) blockIdx.x;
                }
                return false;
            }
        }
    }
    asm volatile("fence.proxy.async.global;" ::: "memory");
    return true;
}

template <bool PAIR, class Last>
__global__ void __launch_bounds__(plane::THREADS, 1)
newton_schulz_kernel(const __grid_constant__ Maps maps, const __grid_constant__ Chain c, const __grid_constant__ typename Last::Args last) {
    using C = plane::Cfg<TERMS, TERMS, PAIR>;
    extern __shared__ uint8_t smem_raw[];
    plane::Engine<Fp16Planes, TERMS, TERMS, PAIR> e;
    e.open(smem_raw, c.status_word);
    const int unit = (int) blockIdx.x / (PAIR ? 2 : 1), units = (int) gridDim.x / (PAIR ? 2 : 1);
    const int products = 3 * c.steps;
    Item w;
    int batch, tm, tn;
    unsigned barriers = 0;  // passed so far
    auto product = [&](int i) -> const Product& { return i % 3 == 0 ? c.gram : i % 3 == 1 ? c.poly : i + 1 < products ? c.apply : c.last; };
    // P and Q have the tiles on and below the diagonal: rows of tile t turn down the columns after it
    auto turn = [&](int which, int t) {
        return which == X_ROWS ? plane::ALONG : which == X_COLUMNS ? plane::DOWN : (t + 1) * (C::TILE_M / plane::BK);
    };
    auto map_of = [&](int which, int i) { return which == P_SYM ? maps.p.m : which == Q_SYM ? maps.q.m : maps.x[i / 3 & 1].m; };

    if (e.warp < 4) {
        plane::few_registers();
        if (e.warp == 0 && e.lane == 0) {
            bool ok = true;
            for (int i = 0; ok && i < products; i++) {
                const Product& g = product(i);
                ok = barriers == 0 || wait_for_count(c.arrived, barriers * gridDim.x, e.abort_flag, c.status_word);
                for (int k = 0; ok && item_at(g, k, unit, units, w); k++) {
                    place(g, w.tile, batch, tm, tn);
                    const plane::Operand a = {map_of(g.a, i), tm * C::TILE_M + (int) e.rank * 128, turn(g.a, tm)};
                    const plane::Operand b = {map_of(g.b, i), tn * C::BN + (int) e.rank * 128, turn(g.b, tn)};
                    ok = e.load(a, b, batch, c.batch, w.kb0, w.kb1);
                }
                barriers += g.cut ? 2 : 1;
            }
            if (!ok || !e.loads_done()) e.drain_loads();
        } else if (e.warp == 1 && e.lane == 0 && e.rank == 0) {
            bool ok = !(c.mute && blockIdx.x == 0);
            for (int i = 0; ok && i < products; i++) {
                const Product& g = product(i);
                for (int k = 0; ok && item_at(g, k, unit, units, w); k++) {
                    place(g, w.tile, batch, tm, tn);
                    ok = e.multiply(turn(g.a, tm), turn(g.b, tn), w.kb0, w.kb1, c.fold);
                }
            }
        }
    } else {
        plane::many_registers();
        const bool leader = threadIdx.x == 128;
        // Once a wait has given up a warp does no more work, but comes to every barrier, so that nobody waits for it; its CTA says so
        // there, and nobody works on, or stores a result, from what it left undone.
        bool ok = true;
        // all drain warps: wait until all CTAs have come to `barriers` barriers
        auto meet = [&]() {
            if (leader) {
                wait_for_count(c.arrived, barriers * gridDim.x, e.abort_flag, c.status_word);
                if (*(volatile unsigned*) (c.arrived + 1)) *e.abort_flag = 1;
            }
            ptx::named_barrier_sync(1, 256);
            ok = __all_sync(0xffffffffu, ok && *e.abort_flag == 0);
        };
        auto arrive = [&]() {
            publish();
            ptx::named_barrier_sync(1, 256);
            if (leader) {
                if (*e.abort_flag) *(volatile unsigned*) (c.arrived + 1) = 1;
                count_in(c.arrived);
            }
            barriers++;
        };
        float sum[C::COLS];
        for (int i = 0; i < products; i++) {
            const Product& g = product(i);
            const int kind = i + 1 == products ? 3 : i % 3;
            if (barriers) meet();
            constexpr int WIDE = C::BN / 32, PER_TILE = (C::TILE_M / 32) * WIDE;  // 32 x 32 blocks of a tile, row by row
            const Planes& out = kind == 0 ? c.p : kind == 1 ? c.q : c.x[(i / 3 + 1) & 1];
            int of = -1;  // the matrix whose factors these are: of the product, and of P and I in Q
            float f = 0, kb = 0, ka = 0;
            auto factors = [&](int batch) {
                if (batch == of) return;
                of = batch;
                const StepExponents s = exponents_of(c.exponents, (int) __ldcg(c.shifts + batch * NORM_BLOCKS), i / 3);
                f = kind == 1 ? c.kc : 1.f;
                f = times_power(f, kind == 0 ? -2 * c.exponents.up : kind == 1 ? 4 * s.x - s.q : s.q + s.x - (kind == 2 ? s.next : c.exponents.up));
                kb = times_power(c.kb, 2 * s.x - s.q);
                ka = times_power(c.ka, -s.q);
            };
            // one body for all products, so that its code is fetched once
            auto finish = [&](const TileAt& at, const float* v) {
                if (at.row >= g.rows || at.col >= g.cols) return;
                if (kind == 3) {
                    plane::by_rows(v, (uint32_t*) e.patch, e.lane, Last::writer(last, at, e.lane, f));
                    return;
                }
                plane::by_eights(v, (uint32_t*) e.patch, e.lane, [&](int r, int col, float* u) {
                    r += at.row;
                    col += at.col;
                    if (r >= out.rows || col >= out.cols) return;
#pragma unroll
                    for (int j = 0; j < 8; j++) u[j] *= f;
                    if (kind == 1) {  // Q = a I + b P + c (P P)
                        float old[8];
                        plane::load8<Fp16Planes>(c.p, at.batch, r, col, old);
#pragma unroll
                        for (int j = 0; j < 8; j++) u[j] += kb * old[j] + (r == col + j ? ka : 0.f);
                    }
                    plane::store8<Fp16Planes, TERMS>(out, at.batch, r, col, u);
                });
            };
            for (int k = 0; ok && item_at(g, k, unit, units, w); k++) {
                TileAt at;
                place(g, w.tile, at.batch, tm, tn);
                factors(at.batch);  // while the tile is multiplied
                ok = e.collect(w.kb0, w.kb1, c.fold, g.K, kind == 0 ? gram_loss() : kind == 1 ? square_loss(c.fold) : no_loss(), sum);
                if (!ok) break;
                const int row = (int) e.rank * plane::BM + e.quarter() * 32;
                at.row = tm * C::TILE_M + row;
                e.blocks(sum, [&](int column, const float* v) {
                    const int b = row / 32 * WIDE + column / 32;
                    at.col = tn * C::BN + column;
                    if (w.slot < 0) finish(at, v);
                    else plane::store_values(c.parts + ((long long) w.slot * PER_TILE + b) * 1024, v, e.lane);
                });
            }
            if (g.cut) {
                arrive();
                meet();
                const int total = g.cut * PER_TILE;
                for (int b = (int) blockIdx.x * plane::DRAIN_WARPS + e.warp - 4; ok && b < total; b += (int) gridDim.x * plane::DRAIN_WARPS) {
                    TileAt at;
                    place(g, g.whole + b / PER_TILE, at.batch, tm, tn);
                    at.row = tm * C::TILE_M + b % PER_TILE / WIDE * 32;
                    at.col = tn * C::BN + b % WIDE * 32;
                    if (at.row >= g.rows || at.col >= g.cols) continue;
                    factors(at.batch);
                    float v[32];
                    plane::join_parts(c.parts, b, total, g.splits, v, e.lane);
                    finish(at, v);
                    __syncwarp();
                }
            }
            if (i + 1 < products) arrive();
        }
    }
    e.close();
}

// ------------------------------------------------------------------ matrices that fit into the shared memory of a cluster

// X of at most 128 rows and 256 columns per CTA of a cluster stays in shared memory from the first step to the last, as planes
// in the layout that the MMAs read; one launch does a whole batch, a cluster per matrix, and memory is touched to read G and
// to write the result.  The grid-wide barriers, stores and loads between products are what small matrices spend their time
// on otherwise (five steps, FP32: 12 x 96 x 960 188 us in the chain above, 70 here; 1 x 64 x 64 119 and 33).
//
// A step of CTA k, which holds the columns X_k:
//     X_k X_k^T on its own; the parts of P are exchanged: every CTA adds up 128 / cluster rows of all parts, in order of the
//     CTAs, and sends them as planes to all;
//     Q = a I + b P + c P P, by every CTA for itself;
//     X_k <- Q X_k, with the planes of X_k read down their columns.
// The sixteen warps share the 128 x 128 results in 32 x 32 blocks; one thread issues the MMAs of a product, all wait for it.
// Products, blocks and the exchange stop at the rows and columns that there are, rounded up to 32.
constexpr int SMALL_THREADS = 512, SMALL_ROWS = 128, SMALL_COLUMNS = 256, SMALL_CLUSTER = 8;
constexpr int SUB_BYTES = 128 * 128;          // 128 rows of 64 values, 128-byte swizzled
constexpr int SQUARE_BYTES = 2 * TERMS * SUB_BYTES;  // planes of 128 x 128 values: [plane][64 columns]
constexpr int HALF_PATCH = 16 * 128;          // 16 rows of 32 FP32
constexpr int SMALL_SMEM = 1024 + 2 * SQUARE_BYTES + SQUARE_BYTES + 16 * HALF_PATCH + MAX_STEPS * 16 + 512;
static_assert(SMALL_SMEM <= plane::MAX_SMEM, "X, P and the patches fit");
static_assert(SQUARE_BYTES + 16 * HALF_PATCH >= 16 * plane::PATCH_FLOATS * 4, "the patches of the result lie where P and the others were");

struct Small {
    int m, n, tall, batch, steps, cluster, slice;  // slice: columns of X per CTA
    float eps, ka, kb, kc;
    Exponents exponents;
    int mute;         // self-test: the first CTA never multiplies
    int* status_word;
};

// byte offset of row r, column c (of 128) in a plane of a square
__device__ __forceinline__ uint32_t square_at(int r, int c) { return (uint32_t) ((c >> 6) * SUB_BYTES + r * 128 + ((((c & 63) >> 3) ^ (r & 7)) << 4) + (c & 7) * 2); }

// 32 consecutive values (columns c0 ...) of row r of a square, from FP32 and back
__device__ __forceinline__ void put_row(uint8_t* square, int r, int c0, const float* value) {
#pragma unroll
    for (int q = 0; q < 4; q++) {
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] = value[8 * q + e];
#pragma unroll
        for (int t = 0; t < TERMS; t++) {
            uint4 o;
            o.x = Fp16Planes::next(v[0], v[1]); o.y = Fp16Planes::next(v[2], v[3]);
            o.z = Fp16Planes::next(v[4], v[5]); o.w = Fp16Planes::next(v[6], v[7]);
            *reinterpret_cast<uint4*>(square + t * 2 * SUB_BYTES + square_at(r, c0 + 8 * q)) = o;
        }
    }
}
__device__ __forceinline__ void get_row(const uint8_t* square, int r, int c0, float* v) {
#pragma unroll
    for (int q = 0; q < 4; q++) {
        const uint4 h = *reinterpret_cast<const uint4*>(square + square_at(r, c0 + 8 * q)), l = *reinterpret_cast<const uint4*>(square + 2 * SUB_BYTES + square_at(r, c0 + 8 * q));
        const uint32_t hi[4] = {h.x, h.y, h.z, h.w}, lo[4] = {l.x, l.y, l.z, l.w};
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const float2 a = Fp16Planes::value(hi[e]), b = Fp16Planes::value(lo[e]);
            v[8 * q + 2 * e] = fmaf(b.x, 1.f / Fp16Planes::TERM, a.x);
            v[8 * q + 2 * e + 1] = fmaf(b.y, 1.f / Fp16Planes::TERM, a.y);
        }
    }
}

// D(main) + D(main2) = A B, D(cross) (+)= its two smaller products: squares a and b, b along its rows or down its columns; n columns of
// the result, `depth` of K, both multiples of 32.  main2 takes what is beyond the first 64 of K, or is main.
__device__ __forceinline__ void square_product(uint32_t main, uint32_t main2, uint32_t cross, uint32_t a, uint32_t b, bool down, bool more, int n, int depth) {
    const uint32_t idesc = plane::idesc_16(Fp16Planes::FORMAT, 128, n) | (down ? 1u << 16 : 0u);
    // down: 64 columns further is a sub-tile (leading offset), 16 rows of K are 2048 bytes; along: 16 of K are 32 bytes, 64 a sub-tile
    const uint64_t da = ptx::make_kmajor_sw128_desc(a), db = ptx::make_kmajor_sw128_desc(b) + (down ? (uint64_t) ((SUB_BYTES >> 4) - 1) << 16 : 0);
    uint32_t again = 0;
#pragma unroll 1
    for (int k = 0; k < depth / 16; k++) {
        const uint32_t ka = (uint32_t) ((k >> 2) * SUB_BYTES + (k & 3) * 32) >> 4, kb = down ? (uint32_t) (k * 2048) >> 4 : ka;
        const uint32_t plane = 2 * SUB_BYTES >> 4, first = more || k > 0;
        plane::umma<false>(cross, da + plane + ka, db + kb, idesc, first);
        plane::umma<false>(cross, da + ka, db + plane + kb, idesc, 1u);
        plane::umma<false>(main, da + ka, db + kb, idesc, again);
        again = 1;
        if (k == 3 && main2 != main) {
            main = main2;
            again = 0;
        }
    }
}

__device__ __forceinline__ uint32_t remote(uint32_t local, int rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(local), "r"(rank));
    return r;
}

template <typename T, class Last>
__global__ void __launch_bounds__(SMALL_THREADS, 1)
small_kernel(const Source<T> s, const Small p, const typename Last::Args last) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t* x = (uint8_t*) (((uintptr_t) smem_raw + 1023) & ~(uintptr_t) 1023);  // one or two squares
    uint8_t* square = x + 2 * SQUARE_BYTES;                                     // P, Q, and the parts of P
    uint8_t* patches = square + SQUARE_BYTES;
    float4* factors = (float4*) (patches + 16 * HALF_PATCH);                    // of every step: of P P, P and I in Q, and of Q X
    double* sums = (double*) (factors + MAX_STEPS);                             // per warp, then per CTA
    uint64_t* bar = (uint64_t*) (sums + 32);
    uint32_t* tmem_slot = (uint32_t*) (bar + 1);
    volatile int* abort_flag = (volatile int*) (tmem_slot + 1);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = p.cluster > 1 ? (int) ptx::cluster_ctarank() : 0, batch = (int) blockIdx.x / p.cluster;
    const int c0 = rank * p.slice, columns = min(p.slice, p.n - c0), squares = p.slice > 128 ? 2 : 1;
    const uint32_t done = ptx::smem_u32(bar);
    auto meet = [&]() {  // all CTAs of the cluster
        if (p.cluster > 1) ptx::cluster_sync_all();
        else __syncthreads();
    };

    if (threadIdx.x == 0) {
        ptx::mbar_init(done, 1);
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 0) ptx::tmem_alloc<false>(ptx::smem_u32(tmem_slot), 512);
    if (threadIdx.x >= SMALL_THREADS - MAX_STEPS) {  // fetched while G is: the bounds that the steps' factors are made of
        const int step = threadIdx.x - (SMALL_THREADS - MAX_STEPS);
        factors[step] = make_float4(0.f, (float) p.exponents.q[step], (float) p.exponents.x[step + 1], 0.f);
    }
    // the source: X's columns [c0, c0 + columns) are eights along rows of G, or rows of G where X is its transpose
    const int lines = p.tall ? columns : p.m, eights = ((p.tall ? p.m : columns) + 7) / 8, row0 = p.tall ? c0 : 0, col0 = p.tall ? 0 : c0;
    double sum = 0;
    for (int i = threadIdx.x; i < lines * eights; i += SMALL_THREADS) {
        const int r = i / eights, c = (i - r * eights) * 8;
        float v[8];
        source8<T, true>(s, batch, row0 + r, col0 + c, v);
        const int have = min(8, (p.tall ? p.m : columns) - c);  // the last eight may reach into the next CTA's columns
#pragma unroll
        for (int e = 0; e < 8; e++)
            if (e < have) sum += (double) v[e] * v[e];
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) sums[warp] = sum;
    for (uint4* z = (uint4*) x + threadIdx.x; z < (uint4*) (x + squares * SQUARE_BYTES); z += SMALL_THREADS) *z = make_uint4(0, 0, 0, 0);
    ptx::tcgen05_fence_before();
    meet();
    ptx::tcgen05_fence_after();
    if (threadIdx.x < p.cluster) {
        sum = 0;
        for (int w = 0; w < 16; w++) sum += sums[w];
        asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(remote(ptx::smem_u32(sums + 16 + rank), (int) threadIdx.x)), "d"(sum) : "memory");
    }
    meet();
    sum = 0;
    for (int k = 0; k < p.cluster; k++) sum += sums[16 + k];
    int shift;
    const double inverse = first_factor(sqrt(sum), p.eps, p.exponents.up, shift);
    const uint32_t tmem = *tmem_slot;
    if (threadIdx.x == SMALL_THREADS - 1) {  // there before the first product ends
        StepExponents e;
        begin(p.exponents, shift, e);
        for (int step = 0; step < p.steps; step++) {
            const float4 bounds = factors[step];
            advance(p.exponents, (int) bounds.y, (int) bounds.z, e);
            factors[step] = make_float4(times_power(p.kc, 4 * e.x - e.q), times_power(p.kb, 2 * e.x - e.q), times_power(p.ka, -e.q),
                                        times_power(1.f, e.q + e.x - (step + 1 < p.steps ? e.next : p.exponents.up)));
        }
    }

    for (int i = threadIdx.x; i < lines * eights; i += SMALL_THREADS) {
        const int r = i / eights, c = (i - r * eights) * 8;
        const int have = min(8, (p.tall ? p.m : columns) - c);
        float v[8];
        source8<T, false>(s, batch, row0 + r, col0 + c, v);
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] = e < have ? (float) ((double) v[e] * inverse) : 0.f;
        if (!p.tall) {
            uint8_t* to = x + (c >> 7) * SQUARE_BYTES + square_at(r, c & 127);
#pragma unroll
            for (int t = 0; t < TERMS; t++) {
                uint4 o;
                o.x = Fp16Planes::next(v[0], v[1]); o.y = Fp16Planes::next(v[2], v[3]);
                o.z = Fp16Planes::next(v[4], v[5]); o.w = Fp16Planes::next(v[6], v[7]);
                *reinterpret_cast<uint4*>(to + t * 2 * SUB_BYTES) = o;
            }
        } else {
#pragma unroll
            for (int t = 0; t < TERMS; t++) {
#pragma unroll
                for (int e = 0; e < 8; e += 2) {
                    const uint32_t o = Fp16Planes::next(v[e], v[e + 1]);
                    uint8_t* to = x + (r >> 7) * SQUARE_BYTES + t * 2 * SUB_BYTES;
                    if (e < have) *reinterpret_cast<uint16_t*>(to + square_at(c + e, r & 127)) = (uint16_t) o;
                    if (e + 1 < have) *reinterpret_cast<uint16_t*>(to + square_at(c + e + 1, r & 127)) = (uint16_t) (o >> 16);
                }
            }
        }
    }

    const int quarter = warp & 3, wide = (warp >> 2) * 32;            // this warp's block of a square: rows and columns
    const uint32_t lanes = (uint32_t) (quarter * 32) << 16;
    const int row = quarter * 32 + lane;
    const int m32 = (p.m + 31) / 32 * 32;
    const bool in_square = quarter * 32 < m32 && wide < m32;
    auto width = [&](int q) { return min(128, (columns - 128 * q + 31) / 32 * 32); };  // of a square of X; nothing or less: none
    // room for the parts: the second square of X if there is none, else the place of P and Q, which then needs two more meetings
    const bool apart = squares == 1;
    uint8_t* parts = apart ? x + SQUARE_BYTES : square;
    uint32_t phase = 0;
    // shared memory that this thread wrote is there for the MMAs of all; then one thread issues them and all wait
    auto multiply = [&](auto issue) {
        ptx::fence_proxy_async_smem();
        ptx::tcgen05_fence_before();
        __syncthreads();
        if (threadIdx.x == 0 && !(p.mute && blockIdx.x == 0)) {
            ptx::tcgen05_fence_after();
            issue();
            ptx::umma_commit(done);
        }
        if (!ptx::mbar_wait(done, phase, abort_flag, p.status_word, 560))  // all CTAs of the cluster work on, but none stores a result
            for (int k = 0; k < p.cluster; k++)
                asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(remote(ptx::smem_u32((const void*) abort_flag), k)), "r"(1) : "memory");
        __syncwarp();
        phase ^= 1;
        ptx::tcgen05_fence_after();
    };
    auto read = [&](uint32_t column, float* v) {
        ptx::tmem_ld32(tmem + lanes + column + (uint32_t) wide, v);
        ptx::tmem_ld_wait();
    };

    // What is beyond 64 of K is added up apart, in columns 256 and on, for four truncated additions each; not in the sum of two squares
    // of X, which take 128 of K each there.
    auto read_two = [&](uint32_t column, bool two, float up, float up2, float* v, float* u) {
        read(column, v);
#pragma unroll
        for (int j = 0; j < 32; j++) v[j] *= up;
        if (!two) return;
        read(column + 256, u);
#pragma unroll
        for (int j = 0; j < 32; j++) v[j] = fmaf(u[j], up2, v[j]);
    };
    const int first = apart ? 64 : 128;  // columns of X whose squares are summed first
    const float f = times_power(1.f, -2 * p.exponents.up);
    for (int step = 0; step < p.steps; step++) {
        float v[32], u[32];
        // ---- P: main sums of the squares in columns 0 and 256, both squares' smaller products in 128
        multiply([&]() {
            for (int q = 0; q < squares; q++) {
                const uint32_t at = ptx::smem_u32(x + q * SQUARE_BYTES);
                if (width(q) > 0) square_product(tmem + 256 * q, tmem + 256 * (apart ? 1 : q), tmem + 128, at, at, false, q > 0, m32, width(q));
            }
        });
        if (in_square) {
            read_two(0, columns > first, gram_loss().factor(min(columns, first)), gram_loss().factor(columns - first), v, u);
            read(128, u);
#pragma unroll
            for (int j = 0; j < 32; j++) v[j] = f * fmaf(u[j], 1.f / Fp16Planes::TERM, v[j]);
            if (p.cluster == 1) put_row(square, row, wide, v);
        }
        if (p.cluster > 1) {
            const int own = m32 / p.cluster;  // rows that a CTA adds up
            if (!apart) meet();               // nobody needs its Q any more
            if (in_square) {                  // parts are [CTA][row][128]
                float* patch = (float*) (patches + warp * HALF_PATCH);
#pragma unroll
                for (int h = 0; h < 2; h++) {  // sixteen rows at a time through the patch, so that remote stores are whole lines
                    if ((lane >> 4) == h) {
#pragma unroll
                        for (int j = 0; j < 8; j++)
                            *reinterpret_cast<float4*>(patch + (lane & 15) * 32 + 4 * (j ^ (lane & 7))) = make_float4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
                    }
                    __syncwarp();
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const int r = 4 * i + (lane >> 3), to = quarter * 32 + 16 * h + r, owner = to / own;
                        const float4 o = *reinterpret_cast<const float4*>(patch + r * 32 + 4 * ((lane & 7) ^ (r & 7)));
                        const uint32_t at = remote(ptx::smem_u32(parts) + (uint32_t) (((rank * own + to - owner * own) * 128 + wide + 4 * (lane & 7)) * 4), owner);
                        asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(at), "f"(o.x), "f"(o.y), "f"(o.z), "f"(o.w) : "memory");
                    }
                    __syncwarp();
                }
            }
            meet();
            constexpr int TURNS = SMALL_ROWS / 2 * 32 / SMALL_THREADS;  // four values of a row each; two CTAs are the fewest that share
            float4 mine[TURNS];
#pragma unroll
            for (int q = 0; q < TURNS; q++) {
                const int i = q * SMALL_THREADS + threadIdx.x;
                if (i >= own * 32 || i % 32 * 4 >= m32) continue;
                const float4* part = (const float4*) parts + i;
                mine[q] = part[0];
                for (int k = 1; k < p.cluster; k++) {
                    const float4 o = part[k * own * 32];
                    mine[q].x += o.x; mine[q].y += o.y; mine[q].z += o.z; mine[q].w += o.w;
                }
            }
            if (!apart) meet();  // all parts have been read: P takes their place
#pragma unroll
            for (int q = 0; q < TURNS; q++) {
                const int i = q * SMALL_THREADS + threadIdx.x, r = rank * own + i / 32, c = i % 32 * 4;
                if (i >= own * 32 || c >= m32) continue;
                float e[4] = {mine[q].x, mine[q].y, mine[q].z, mine[q].w};
#pragma unroll
                for (int t = 0; t < TERMS; t++) {
                    const uint32_t a = Fp16Planes::next(e[0], e[1]), b = Fp16Planes::next(e[2], e[3]);
                    const uint32_t at = ptx::smem_u32(square) + (uint32_t) (t * 2 * SUB_BYTES) + square_at(r, c);
                    for (int k = 0; k < p.cluster; k++)
                        asm volatile("st.shared::cluster.v2.b32 [%0], {%1, %2};" ::"r"(remote(at, k)), "r"(a), "r"(b) : "memory");
                }
            }
            asm volatile("fence.proxy.async;" ::: "memory");
            meet();
        }
        // ---- Q, in place of P
        const uint32_t sq = ptx::smem_u32(square);
        multiply([&]() { square_product(tmem, tmem + 256, tmem + 128, sq, sq, false, false, m32, m32); });
        if (in_square) {
            read_two(0, m32 > 64, square_loss(1).factor(min(p.m, 64)), square_loss(1).factor(p.m - 64), v, u);
            read(128, u);
#pragma unroll
            for (int j = 0; j < 32; j++) v[j] = fmaf(u[j], 1.f / Fp16Planes::TERM, v[j]);
            get_row(square, row, wide, u);
            const float4 k = factors[step];
#pragma unroll
            for (int j = 0; j < 32; j++) v[j] = k.x * v[j] + k.y * u[j] + (row == wide + j && row < p.m ? k.z : 0.f);
            put_row(square, row, wide, v);
        }
        // ---- X, a square at a time; in the last step at once, as the patches of the result lie where Q is
        const float apply = factors[step].w;
        const bool at_once = squares == 2 && step + 1 == p.steps;
        for (int q = 0; q < squares; q++) {
            const uint32_t to = at_once ? 256 * q : 0;
            if (q == 0 || !at_once)
                multiply([&]() {
                    for (int i = q; i < (at_once ? 2 : q + 1); i++)
                        if (width(i) > 0)
                            square_product(tmem + (at_once ? 256 * i : 0), tmem + (at_once ? 256 * i : 256), tmem + (at_once ? 256 * i : 0) + 128, sq,
                                           ptx::smem_u32(x + i * SQUARE_BYTES), true, false, width(i), m32);
                });
            if (q == 0 && step + 1 == p.steps) {
                meet();
                if (*abort_flag) break;
            }
            if (quarter * 32 >= m32 || wide >= width(q)) continue;
            read_two(to, !at_once && m32 > 64, 1.f, 1.f, v, u);
            read(to + 128, u);
#pragma unroll
            for (int j = 0; j < 32; j++) v[j] = fmaf(u[j], 1.f / Fp16Planes::TERM, v[j]);
            if (step + 1 < p.steps) {
#pragma unroll
                for (int j = 0; j < 32; j++) v[j] *= apply;
                put_row(x + q * SQUARE_BYTES, row, wide, v);
            } else {
                const int column = c0 + q * 128 + wide;
                TileAt at;
                at.batch = batch;
                at.row = p.tall ? column : quarter * 32;
                at.col = p.tall ? quarter * 32 : column;
                const int end = c0 + columns;  // the columns after them are another CTA's
                if (p.tall) {
                    const auto write = Last::writer(last, at, lane, apply);
#pragma unroll
                    for (int j = 0; j < 32; j++)
                        if (column + j < end) write(j, v[j]);
                } else {
                    auto write = Last::writer(last, at, lane, apply);
                    if (column + lane >= end) write.rows = 0;
                    plane::by_rows(v, (uint32_t*) square + warp * plane::PATCH_FLOATS, lane, write);
                    __syncwarp();
                }
            }
        }
    }
    ptx::tcgen05_fence_before();
    meet();
    if (warp == 0) {
        if (*abort_flag) {  // products that nobody waited for come to their end
            const unsigned long long t0 = ptx::global_ns();
            while ((long long) (ptx::global_ns() - t0) < 20000000LL) __nanosleep(1000);
        }
        ptx::tcgen05_fence_after();
        ptx::tmem_free<false>(tmem, 512);
    }
}

// ------------------------------------------------------------------ host side

int bad(const char* who, const char* what) {
    set_error("%s: %s", who, what);
    return CAKEB200_ERR_ARG;
}

constexpr int MAX_SIDE = 1 << 20, MAX_BATCH = 65535;
thread_local int g_mute = 0;  // in a self-test's call

struct Layout {
    Planes x[2], p, q;
    double* partial;
    unsigned* arrived;
    float* parts;
    size_t bytes;
};

// The products of one matrix size for one form.  Returns the time of a step.
double plan(Product* gram, Product* poly, Product* apply, Product* last, int m, int n, bool tall, int batch, bool pair, int units) {
    gram->a = gram->b = X_ROWS;
    poly->a = poly->b = P_SYM;
    apply->a = Q_SYM; apply->b = X_COLUMNS;
    // the result as the caller stores it: Q X, or its transpose X^T Q (Q is symmetric)
    last->a = tall ? X_COLUMNS : Q_SYM; last->b = tall ? Q_SYM : X_COLUMNS;
    const plane::Costs costs = plane::costs_of(TERMS, TERMS, 3, 2.2);
    const double t = plane::plan(gram, m, m, n, 1, batch, pair, units, costs) + plane::plan(poly, m, m, m, 1, batch, pair, units, costs) +
                     plane::plan(apply, m, n, m, 0, batch, pair, units, costs);
    plane::plan(last, tall ? n : m, tall ? m : n, m, 0, batch, pair, units, costs);
    return t;
}

// Room for the parts of cut tiles of any product, in either form.
size_t parts_bytes(int m, int n, int batch) {
    size_t most = 0;
    for (int pair = 0; pair < 2; pair++) {
        const int side = pair ? 256 : 128;
        const long long bm = (m + plane::BK - 1) / plane::BK, bn = (n + plane::BK - 1) / plane::BK;
        const long long pieces = std::max(plane::count_tiles(m, m, batch, true, side) * std::max(bm, bn), plane::count_tiles(m, n, batch, false, side) * bm);
        most = std::max(most, plane::parts_bytes(pieces, pair != 0));
    }
    return most;
}
Layout lay_out(char* base, int batch, int m, int n) {
    Layout l;
    size_t at = 0;
    auto planes = [&](int rows, int cols) {
        Planes p;
        p.base = (uint16_t*) (base + at);
        p.rows = rows; p.cols = cols; p.ld = plane::padded(cols); p.batches = batch;
        at += plane::plane_bytes(TERMS, batch, rows, cols);
        return p;
    };
    l.x[0] = planes(m, n);
    l.x[1] = planes(m, n);
    l.p = planes(m, m);
    l.q = planes(m, m);
    l.partial = (double*) (base + at);
    at += ((size_t) batch * NORM_BLOCKS * 8 + 1023) / 1024 * 1024;
    l.arrived = (unsigned*) (base + at);
    at += 1024;
    l.parts = (float*) (base + at);
    at += parts_bytes(m, n, batch);
    l.bytes = at;
    return l;
}

int check_shape(const char* who, int rows, int cols, int batch) {
    if (rows <= 0 || cols <= 0 || batch < 0) return bad(who, "sizes must be positive");
    if (rows > MAX_SIDE || cols > MAX_SIDE || batch > MAX_BATCH) {
        set_error("%s: more than 2^20 rows or columns, or 65535 matrices", who);
        return CAKEB200_ERR_TOO_LARGE;
    }
    return CAKEB200_OK;
}

// Whether two matrices of `rows` rows share memory: addresses, bytes of a row, bytes from row to row.  Rows of the same pitch may lie
// beside one another.
bool overlap(const void* a, long long width_a, long long pitch_a, const void* b, long long width_b, long long pitch_b, int rows) {
    const long long from_a = (long long) (uintptr_t) a, from_b = (long long) (uintptr_t) b;
    if (from_a + (rows - 1) * pitch_a + width_a <= from_b || from_b + (rows - 1) * pitch_b + width_b <= from_a) return false;
    if (pitch_a != pitch_b) return true;
    const long long d = ((from_b - from_a) % pitch_a + pitch_a) % pitch_a;
    return d < width_a || d + width_b > pitch_a;
}

struct Coefficients {
    int steps;
    float a, b, c, eps;
};

// the exponent e of the first power of two at or above v >= 0
short exponent_above(double v) {
    if (!(v > 0)) return FAR_BELOW;
    if (!std::isfinite(v)) return -FAR_BELOW;
    return (short) std::ceil(std::log2(v) - 1e-6);  // a bound that its own rounding put above a power of two is that power
}
// An X whose singular values are all about 1 / sqrt(m) has elements around 1 as it is held, and 2^-12 of that is the least that FP16 pairs
// hold with all their bits.  So coefficients may let a singular value of 1 grow 2^12 times as far as small ones, which grow by |a| a step;
// where it would run away further the bounds are those of singular values up to 2, and larger ones come out infinite.
Exponents exponents_for(const Coefficients& k, int up, bool runaway = false) {
    Exponents e = {};
    double small = 1;
    e.up = (short) up;
    const double a = k.a, b = k.b, c = k.c;
    e.a = exponent_above(std::fabs(a)); e.b = exponent_above(std::fabs(b)); e.c = exponent_above(std::fabs(c));
    double u = 1;  // the largest singular value so far
    for (int s = 0; s < k.steps; s++) {
        const double y = u * u;
        auto quotient = [&](double t2) { return std::fabs(a + b * t2 + c * t2 * t2); };
        // their extremes over [0, u]: the ends, and where the derivative is zero (of b t^2 + c t^4; of a t + b t^3 + c t^5)
        double q = std::max(quotient(0), quotient(y)), x = u * quotient(y);
        if (c != 0) {
            const double t2 = -b / (2 * c), d = 9 * b * b - 20 * a * c;
            if (t2 > 0 && t2 < y) q = std::max(q, quotient(t2));
            if (d >= 0)
                for (double root : {std::sqrt(d), -std::sqrt(d)}) {
                    const double r2 = (root - 3 * b) / (10 * c);
                    if (r2 > 0 && r2 < y) x = std::max(x, std::sqrt(r2) * quotient(r2));
                }
        } else if (b != 0) {
            const double r2 = -a / (3 * b);
            if (r2 > 0 && r2 < y) x = std::max(x, std::sqrt(r2) * quotient(r2));
        }
        e.x[s] = exponent_above(u);
        e.q[s] = exponent_above(q);
        if (!runaway && u > 4096 * small) return exponents_for(k, up, true);
        u = runaway ? std::min(x, 2.0) : x;
        small *= std::fabs(a);
    }
    e.x[k.steps] = exponent_above(u);
    return e;
}

int check_coefficients(const char* who, const Coefficients& k) {
    if (k.steps < 1 || k.steps > MAX_STEPS) return bad(who, "1 to 64 steps");
    if (!(k.eps >= 0.f)) return bad(who, "eps is a number that is not negative");
    if (!std::isfinite(k.a) || !std::isfinite(k.b) || !std::isfinite(k.c)) return bad(who, "the coefficients are finite numbers");
    return CAKEB200_OK;
}

template <typename T>
Matrix<T> matrix(T* base, long long ld, long long stride, int rows, int batch) {
    Matrix<T> m;
    m.base = base;
    m.ld = ld;
    m.stride = stride;
    m.vec = (uintptr_t) base % 16 == 0 && (rows == 1 || ld * (long long) sizeof(T) % 16 == 0) && (batch == 1 || stride * (long long) sizeof(T) % 16 == 0);
    return m;
}

// A kernel that may be set up while the one before it ends.
template <typename... P, typename... A>
int launch_after(void (*kernel)(P...), dim3 grid, cudaStream_t s, const A&... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(256);
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    CAKE_CUDA_OK(cudaLaunchKernelEx(&cfg, kernel, P(args)...));
    return CAKEB200_OK;
}

// Units of one form that are resident together on the current device (asked once per device and kernel).
template <bool PAIR, class Last>
int resident_units(int* out) {
    using C = plane::Cfg<TERMS, TERMS, PAIR>;
    auto kernel = newton_schulz_kernel<PAIR, Last>;
    static std::atomic<int> known[64];
    int dev = 0;
    CAKE_CUDA_OK(cudaGetDevice(&dev));
    if (dev < 64 && (*out = known[dev].load()) > 0) return CAKEB200_OK;
    CAKE_CUDA_OK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM));
    int n = 0;
    if (PAIR) {
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(2);
        cfg.blockDim = dim3(plane::THREADS);
        cfg.dynamicSmemBytes = C::SMEM;
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = 2;
        attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        CAKE_CUDA_OK(cudaOccupancyMaxActiveClusters(&n, kernel, &cfg));
    } else {
        int per_sm = 0, sms = 0;
        CAKE_CUDA_OK(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kernel, plane::THREADS, C::SMEM));
        CAKE_CUDA_OK(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev));
        n = per_sm * sms;
    }
    n = std::min(n, PAIR ? plane::MAX_UNITS / 2 : plane::MAX_UNITS);
    if (n < 1) {
        set_error("the orthogonalisation kernel does not fit the device");
        return CAKEB200_ERR_CUDA;
    }
    if (dev < 64) known[dev] = n;
    *out = n;
    return CAKEB200_OK;
}

template <bool PAIR, class Last>
int launch_chain(const Maps& maps, const Chain& c, const typename Last::Args& last, int units, cudaStream_t s) {
    using C = plane::Cfg<TERMS, TERMS, PAIR>;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned) (PAIR ? 2 * units : units));
    cfg.blockDim = dim3(plane::THREADS);
    cfg.dynamicSmemBytes = C::SMEM;
    cfg.stream = s;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeCooperative;
    attr[0].val.cooperative = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = PAIR ? 2 : 1;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    CAKE_CUDA_OK(cudaLaunchKernelEx(&cfg, newton_schulz_kernel<PAIR, Last>, maps, c, last));
    return CAKEB200_OK;
}

// Whether the matrices fit clusters, and how.
bool fits_small(int m, int n, int batch, int sm_count, Small* p) {
    if (m > SMALL_ROWS || n > SMALL_COLUMNS * SMALL_CLUSTER) return false;
    int c = 1;
    while (c * SMALL_COLUMNS < n) c *= 2;
    // half as many columns per CTA make a step shorter as long as all clusters are resident together
    while (c < SMALL_CLUSTER && n > 128 * c && (long long) batch * 2 * c <= sm_count * 3 / 4) c *= 2;
    // One CTA per matrix is faster than the chain for any batch (2000 of 64 x 128: 0.47 ms, 1.19 in the chain).  Clusters are
    // as long as few wait for others: of 8 CTAs, 128 x 2048, 32 matrices 326 us (chain 326), 48 434 (405), 64 x 1000, 64 matrices 145 (280).
    if (c > 1 && (long long) batch * c > 3ll * sm_count) return false;
    p->cluster = c;  // n > 64 c, so that slices rounded up to 8 leave every CTA some columns
    p->slice = ((n + c - 1) / c + 7) / 8 * 8;
    return true;
}

template <typename T, class Last>
int launch_small(const Source<T>& src, const Small& p, const typename Last::Args& last, int device, cudaStream_t s) {
    const auto kernel = small_kernel<T, Last>;
    static std::atomic<unsigned long long> opted{0};  // devices whose shared-memory limit has been raised for this kernel
    if (device >= 64 || !(opted.load() >> device & 1)) {
        CAKE_CUDA_OK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SMALL_SMEM));
        if (device < 64) opted |= 1ull << device;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned) (p.batch * p.cluster));
    cfg.blockDim = dim3(SMALL_THREADS);
    cfg.dynamicSmemBytes = SMALL_SMEM;
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned) p.cluster;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    CAKE_CUDA_OK(cudaLaunchKernelEx(&cfg, kernel, src, p, last));
    return CAKEB200_OK;
}

// From the source to the last X, which goes through `Last`.
// early: the results of one matrix may be stored while other matrices are still read.
template <typename T, class Last>
int run(const Source<T>& src, int batch, bool early, const Coefficients& k, void* workspace, typename Last::Args last, DeviceState* st, cudaStream_t s) {
    const int rows = src.rows, cols = src.cols;
    const bool tall = rows > cols;
    const int m = tall ? cols : rows, n = tall ? rows : cols;
    // around sqrt(m n), below the 2^16 at which the largest possible element of X would overflow
    const int up = std::min(15, (int) (0.5 * std::log2((double) m * n)));
    const Exponents exponents = exponents_for(k, up);
    int rc, units_single = 0, units_pair = 0;
    Small small = {};
    if (early && option_get(OPT_PAIR) == 0 && option_get(OPT_K_PIECES) == 0 && fits_small(m, n, batch, st->sm_count, &small)) {  // those options are about the chain
        small.m = m; small.n = n; small.tall = tall; small.batch = batch; small.steps = k.steps;
        small.eps = k.eps; small.ka = k.a; small.kb = k.b; small.kc = k.c;
        small.exponents = exponents;
        small.mute = g_mute;
        small.status_word = st->status_word;
        if ((rc = launch_small<T, Last>(src, small, last, st->device, s))) return rc;
        thread_stats()->launches = 1;
        return CAKEB200_OK;
    }
    const Layout l = lay_out((char*) workspace, batch, m, n);
    if ((rc = resident_units<false, Last>(&units_single)) || (rc = resident_units<true, Last>(&units_pair))) return rc;
    const long long tiles = plane::count_tiles(m, n, batch, false, 128);
    if (tiles > (1LL << 27)) {
        set_error("the matrices have too many tiles");
        return CAKEB200_ERR_TOO_LARGE;
    }
    Maps maps;
    if ((rc = plane::encode_planes<Fp16Planes>(maps.x[0].m, l.x[0], TERMS)) || (rc = plane::encode_planes<Fp16Planes>(maps.x[1].m, l.x[1], TERMS)) ||
        (rc = plane::encode_planes<Fp16Planes>(maps.p.m, l.p, TERMS)) || (rc = plane::encode_planes<Fp16Planes>(maps.q.m, l.q, TERMS)))
        return rc;

    Chain c = {};
    c.x[0] = l.x[0]; c.x[1] = l.x[1]; c.p = l.p; c.q = l.q;
    c.batch = batch; c.steps = k.steps; c.fold = fold_for(m);
    c.ka = k.a; c.kb = k.b; c.kc = k.c;
    c.exponents = exponents;
    c.shifts = l.partial + SHIFT_AT;
    c.parts = l.parts;
    c.arrived = l.arrived;
    c.mute = g_mute;
    c.status_word = st->status_word;
    const int forced = option_get(OPT_PAIR);  // 1: pairs, 2: single SMs, 0: the faster by the model
    Chain other = c;
    const double t_single = plan(&c.gram, &c.poly, &c.apply, &c.last, m, n, tall, batch, false, units_single);
    const double t_pair = plan(&other.gram, &other.poly, &other.apply, &other.last, m, n, tall, batch, true, units_pair);
    const bool pair = forced ? forced == 1 : t_pair < t_single;
    if (pair) c = other;
    // no more units than any product gives work to
    int units = 1;
    for (const Product* g : {&c.gram, &c.poly, &c.apply, &c.last}) units = std::max(units, std::max(g->whole, g->cut * g->splits));
    units = std::min(units, pair ? units_pair : units_single);

    const long long work = (long long) rows * ((cols + 7) / 8);
    const int partials = (int) std::max<long long>(1, std::min<long long>(SHIFT_AT, work / 512));
    norm_kernel<T><<<dim3((unsigned) partials, (unsigned) batch), 256, 0, s>>>(src, l.partial);
    CAKE_CUDA_OK(cudaGetLastError());
    const dim3 grid((unsigned) ((cols + 255) / 256), (unsigned) ((rows + 31) / 32), (unsigned) batch);
    if ((rc = launch_after(split_kernel<T>, grid, s, src, l.partial, partials, k.eps, up, tall, l.x[0], l.arrived)))
        return rc;
    rc = pair ? launch_chain<true, Last>(maps, c, last, units, s) : launch_chain<false, Last>(maps, c, last, units, s);
    if (!rc) thread_stats()->launches = 3;
    return rc;
}

bool known(int type) { return type == CAKEB200_F32 || type == CAKEB200_BF16; }

template <typename T>
int orthogonalize(const void* G, long long ldg, long long stride_g, void* out, long long ldo, long long stride_o, int rows, int cols, int batch,
                  const Coefficients& k, void* workspace, DeviceState* st, cudaStream_t s) {
    Source<T> src = {};
    src.g = matrix((const T*) G, ldg, stride_g, rows, batch);
    src.rows = rows;
    src.cols = cols;
    typename ResultEpilogue<T>::Args last = {matrix((T*) out, ldo, stride_o, rows, batch), rows, cols};
    // in place is fine matrix by matrix; a result that lies across its operands has to wait for all of them
    const long long size = sizeof(T), reach_g = (rows - 1) * ldg + cols + (batch - 1) * stride_g, reach_o = (rows - 1) * ldo + cols + (batch - 1) * stride_o;
    const bool same = G == out && ldg == ldo && (batch == 1 || stride_g == stride_o);
    const bool early = batch == 1 || same || (stride_g >= 0 && !overlap(G, reach_g * size, reach_g * size, out, reach_o * size, reach_o * size, 1));
    return run<T, ResultEpilogue<T>>(src, batch, early, k, workspace, last, st, s);
}

template <typename TW, typename TG>
int muon(void* W, long long ldw, const void* G, long long ldg, float* M, long long ldm, int rows, int cols, double lr, double mu, int nesterov,
         double weight_decay, double scale, const Coefficients& k, void* workspace, DeviceState* st, cudaStream_t s) {
    Source<TG> src = {};
    src.g = matrix((const TG*) G, ldg, 0, rows, 1);
    src.m = M;
    src.ldm = ldm;
    src.vec_m = matrix(M, ldm, 0, rows, 1).vec;
    src.mu = (float) mu;
    src.rest = (float) (1.0 - mu);
    src.nesterov = nesterov;
    src.rows = rows;
    src.cols = cols;
    typename StepEpilogue<TW>::Args last = {matrix((TW*) W, ldw, 0, rows, 1), rows, cols, (float) (1.0 - lr * weight_decay), (float) (lr * scale)};
    return run<TG, StepEpilogue<TW>>(src, 1, true, k, workspace, last, st, s);
}

}  // namespace
}  // namespace cakeb200

using namespace cakeb200;

extern "C" {

size_t cakeb200_orthogonalize_workspace(int rows, int cols, int batch, int type) {
    if (check_shape("cakeb200_orthogonalize_workspace", rows, cols, batch)) return 0;
    if (!known(type)) {
        bad("cakeb200_orthogonalize_workspace", "the type is float32 or bfloat16");
        return 0;
    }
    return lay_out(nullptr, batch, std::min(rows, cols), std::max(rows, cols)).bytes;
}

int cakeb200_orthogonalize(const void* G, long long ldg, long long stride_g, void* out, long long ldo, long long stride_o, int rows, int cols,
                           int batch, int type, int steps, float a, float b, float c, float eps, void* workspace, size_t workspace_bytes,
                           void* stream) {
    static const char* who = "cakeb200_orthogonalize";
    *thread_stats() = cakeb200_stats();
    const Coefficients k = {steps, a, b, c, eps};
    int rc = check_shape(who, rows, cols, batch);
    if (rc) return rc;
    if (!known(type)) return bad(who, "the type is float32 or bfloat16");
    if ((rc = check_coefficients(who, k))) return rc;
    if (batch == 0) return CAKEB200_OK;
    if (!G || !out || !workspace) return bad(who, "null pointer");
    if (ldg < cols || ldo < cols) return bad(who, "a leading dimension is smaller than its row");
    if (batch > 1 && stride_o < (long long) (rows - 1) * ldo + cols) return bad(who, "the matrices of the result overlap");
    if ((uintptr_t) workspace % 1024) return bad(who, "the workspace starts on a 1024-byte boundary");
    if (workspace_bytes < cakeb200_orthogonalize_workspace(rows, cols, batch, type)) return bad(who, "the workspace is too small");
    const size_t size = type == CAKEB200_F32 ? 4 : 2;
    if ((uintptr_t) G % size || (uintptr_t) out % size) return bad(who, "a pointer is not aligned to its type");
    DeviceState* st = device_state();
    if (!st) return CAKEB200_ERR_NO_DEVICE;
    if (!on_current_device(G) || !on_current_device(out) || !on_current_device(workspace))
        return bad(who, "operands must be device pointers of the current device");
    cudaStream_t s = (cudaStream_t) stream;
    if (type == CAKEB200_F32) return orthogonalize<float>(G, ldg, stride_g, out, ldo, stride_o, rows, cols, batch, k, workspace, st, s);
    return orthogonalize<__nv_bfloat16>(G, ldg, stride_g, out, ldo, stride_o, rows, cols, batch, k, workspace, st, s);
}

int cakeb200_muon_step(void* W, long long ldw, int type_w, const void* G, long long ldg, int type_g, float* M, long long ldm, int rows, int cols,
                       double lr, double momentum, int nesterov, double weight_decay, double scale, int steps, float a, float b, float c, float eps,
                       void* workspace, size_t workspace_bytes, void* stream) {
    static const char* who = "cakeb200_muon_step";
    *thread_stats() = cakeb200_stats();
    const Coefficients k = {steps, a, b, c, eps};
    int rc = check_shape(who, rows, cols, 1);
    if (rc) return rc;
    if (!known(type_w) || !known(type_g)) return bad(who, "the types are float32 or bfloat16");
    if ((rc = check_coefficients(who, k))) return rc;
    if (!W || !G || !M || !workspace) return bad(who, "null pointer");
    if (ldw < cols || ldg < cols || ldm < cols) return bad(who, "a leading dimension is smaller than its row");
    if ((uintptr_t) workspace % 1024) return bad(who, "the workspace starts on a 1024-byte boundary");
    if (workspace_bytes < cakeb200_orthogonalize_workspace(rows, cols, 1, type_w)) return bad(who, "the workspace is too small");
    if ((uintptr_t) W % (type_w == CAKEB200_F32 ? 4 : 2) || (uintptr_t) G % (type_g == CAKEB200_F32 ? 4 : 2) || (uintptr_t) M % 4)
        return bad(who, "a pointer is not aligned to its type");
    const long long size_w = type_w == CAKEB200_F32 ? 4 : 2, size_g = type_g == CAKEB200_F32 ? 4 : 2;
    if (overlap(M, cols * 4LL, ldm * 4, W, cols * size_w, ldw * size_w, rows) || overlap(M, cols * 4LL, ldm * 4, G, cols * size_g, ldg * size_g, rows))
        return bad(who, "M overlaps W or G");
    DeviceState* st = device_state();
    if (!st) return CAKEB200_ERR_NO_DEVICE;
    if (!on_current_device(W) || !on_current_device(G) || !on_current_device(M) || !on_current_device(workspace))
        return bad(who, "operands must be device pointers of the current device");
    cudaStream_t s = (cudaStream_t) stream;
    nesterov = nesterov ? 1 : 0;
#define CAKE_MUON(TW, TG) \
    return muon<TW, TG>(W, ldw, G, ldg, M, ldm, rows, cols, lr, momentum, nesterov, weight_decay, scale, k, workspace, st, s)
    if (type_w == CAKEB200_F32) {
        if (type_g == CAKEB200_F32) CAKE_MUON(float, float);
        CAKE_MUON(float, __nv_bfloat16);
    }
    if (type_g == CAKEB200_F32) CAKE_MUON(__nv_bfloat16, float);
    CAKE_MUON(__nv_bfloat16, __nv_bfloat16);
#undef CAKE_MUON
}

int cakeb200_selftest_orthogonalize_wait(float* W, const float* G, float* M, int rows, int cols, void* workspace, size_t workspace_bytes,
                                         void* stream) {
    g_mute = 1;
    const int rc = cakeb200_muon_step(W, cols, CAKEB200_F32, G, cols, CAKEB200_F32, M, cols, rows, cols, 1.0, 0.0, 0, 0.0, 1.0, 5, 3.4445f, -4.7750f,
                                      2.0315f, 1e-7f, workspace, workspace_bytes, stream);
    g_mute = 0;
    if (rc) return rc;
    DeviceState* st = device_state();
    return st ? wait_and_check(st, (cudaStream_t) stream) : CAKEB200_ERR_NO_DEVICE;
}

}  // extern "C"
