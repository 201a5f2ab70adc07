// Products with 4-bit weights and many rows: a prompt, or a training batch.
//
// From some tens of rows on the product is no longer bound by reading the codes but by multiplying: rows * N * K multiply-adds
// on tcgen05.  The weights are expanded to bf16 planes (plane_gemm.cuh) in a workspace, a slab of at most 2^25 of them at
// a time, so that they stay in L2 until they have been multiplied; the expansion reads half a byte and writes two to four
// bytes per weight, once per slab whatever the number of rows.
//
// Planes per operand, by the type of x and y:
//   BF16  x as it is, two planes of w (exactly).  Two MMAs per step.  w rounded to a single plane would cost 2^-9 of every
//         product, as much again as the result's own rounding (error 2.4e-3 instead of 1.7e-3), and give a row other results
//         alone than in a batch.  500 x 4096 x 4096 takes 51 us; 39 with a single plane.
//   FP16  two planes each (both exactly): single FP16 planes could not hold every scale.  Three MMAs; the product of the
//         second planes, below 2^-14 of the first ones', is left out.
//   FP32  three planes of x (exactly), two of w (exactly: a 16-bit scale times a whole number below 16).  Five MMAs.
// The gradient for the input reads the same planes of W down their columns.
#include <algorithm>

#include "plane_gemm.cuh"
#include "q4.cuh"

namespace cakeb200 {

using plane::Bf16Planes;
using plane::Planes;
using plane::TileAt;

namespace {

constexpr long long SLAB = 1LL << 25;  // weights expanded at a time

template <typename T> struct Terms;
template <> struct Terms<__nv_bfloat16> { static constexpr int X = 1, W = 2, PRODUCTS = 2, CHUNK = 16; };
template <> struct Terms<__half> { static constexpr int X = 2, W = 2, PRODUCTS = 3, CHUNK = 16; };
template <> struct Terms<float> { static constexpr int X = 3, W = 2, PRODUCTS = 5, CHUNK = 2; };

// Rows [16 rt0, ...) and features [64 kb0, ...) of the weights as planes: a thread per lane of a block, 8 weights to a store.
template <int T>
__global__ void __launch_bounds__(256)
expand_kernel(const Q4View w, int rt0, int rts, int kb0, int kbs, const Planes out) {
    const long long i = (long long) blockIdx.x * 256 + threadIdx.x;
    if (i >= (long long) rts * kbs * 32) return;
    const int lane = (int) (i & 31), a = lane >> 2, t = lane & 3;
    const int block = (int) (i >> 5), kb = block % kbs, rt = block / kbs;
    const uint4 c = __ldg(w.codes + ((long long) (rt0 + rt) * w.steps * 2 + kb0 + kb) * 32 + lane);
    const uint32_t words[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
    for (int h = 0; h < 2; h++) {
        const long long at = q4_scale_at(w, rt0 + rt, (kb0 + kb) >> 1) + q4_scale_place(a, ((kb0 + kb) & 1) * 64 + h * 32, w.group_shift);
        const uint32_t pair = __ldg(reinterpret_cast<const uint32_t*>(w.scales + at));
        const uint32_t z = w.zeros ? __ldg(reinterpret_cast<const uint16_t*>(w.zeros + at)) : 0x0808u;
        const int k = kb * 64 + h * 32 + t * 8;
        if (k >= out.cols) continue;
#pragma unroll
        for (int half = 0; half < 2; half++) {  // rows a and a + 8
            const int r = rt * 16 + a + 8 * half;
            if (r >= out.rows) continue;
            const float s = q4_scale((uint16_t) (pair >> (16 * half)), w.scale_bf16);
            const float zero = (float) ((z >> (8 * half)) & 15u);
            float v[8];
#pragma unroll
            for (int e = 0; e < 8; e++) {  // feature e: word 2 h + e / 4, register 2 (e % 4 / 2) + half, half e % 2 of it
                const uint32_t q = words[2 * h + (e >> 2)] >> (4 * (((e >> 1) & 1) * 2 + half) + 16 * (e & 1)) & 15u;
                v[e] = s * ((float) q - zero);
            }
            plane::store8<Bf16Planes, T>(out, 0, r, k, v);
        }
    }
}

// x (or dy) as planes, eight values per thread.
template <typename T, int TERMS>
__global__ void __launch_bounds__(256)
split_rows_kernel(const T* __restrict__ x, long long ld, int rows, int cols, int vec, const Planes out) {
    const int segments = (cols + 7) / 8;
    const long long i = (long long) blockIdx.x * 256 + threadIdx.x;
    if (i >= (long long) rows * segments) return;
    const int r = (int) (i / segments), c = (int) (i - (long long) r * segments) * 8;
    const T* p = x + r * ld + c;
    float v[8];
    if (vec && c + 8 <= cols) {
        alignas(16) T u[8];
#pragma unroll
        for (int q = 0; q < (int) sizeof(u) / 16; q++) reinterpret_cast<uint4*>(u)[q] = __ldg(reinterpret_cast<const uint4*>(p) + q);
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] = to_float(u[e]);
    } else {
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] = c + e < cols ? to_float(p[e]) : 0.f;
    }
    uint32_t words[4][TERMS];
#pragma unroll
    for (int e = 0; e < 4; e++) split_pair<TERMS>(v[2 * e], v[2 * e + 1], words[e]);
    uint16_t* at = out.base + (long long) r * out.ld + c;
#pragma unroll
    for (int t = 0; t < TERMS; t++)
        *reinterpret_cast<uint4*>(at + (long long) t * out.rows * out.ld) = make_uint4(words[0][t], words[1][t], words[2][t], words[3][t]);
}

// y = D + bias, rounded once
template <typename T>
struct RowsEpilogue {
    struct Args {
        T* out;
        long long ld;
        int rows, cols;
        const T* bias;
        int vec;      // 16-byte stores allowed
    };
    static __device__ __forceinline__ void block(const Args& a, const TileAt& at, const float* v, uint32_t* patch, int lane) {
        plane::by_eights(v, patch, lane, [&](int r, int c, float* u) {
            r += at.row;
            c += at.col;
            if (r >= a.rows || c >= a.cols) return;
            const int n = min(8, a.cols - c);
            if (a.bias) {
#pragma unroll
                for (int e = 0; e < 8; e++)
                    if (e < n) u[e] += to_float(a.bias[c + e]);
            }
            T* p = a.out + r * a.ld + c;
            alignas(16) T o[8];
#pragma unroll
            for (int e = 0; e < 8; e++) o[e] = from_float<T>(u[e]);
            if (a.vec && n == 8) {
#pragma unroll
                for (int q = 0; q < (int) sizeof(o) / 16; q++) reinterpret_cast<uint4*>(p)[q] = reinterpret_cast<const uint4*>(o)[q];
            } else {
#pragma unroll
                for (int e = 0; e < 8; e++)
                    if (e < n) p[e] = o[e];
            }
        });
    }
};

// The slab of weights multiplied at a time: of the result's columns, i.e. output features, or input features of the gradient.
int slab_columns(const Q4View& w, bool dx) {
    const int cols = dx ? w.K : w.N, depth = dx ? w.N : w.K;
    const long long fit = SLAB / plane::padded(depth) / 256 * 256;
    return (int) std::min<long long>(cols, std::max<long long>(fit, 256));
}

struct Room {
    Planes x, w;
    float* parts;
    bool cut;       // tiles may be cut along K, their parts stored
    size_t bytes;
};

template <typename T>
Room lay_out(char* base, const Q4View& w, int rows, bool dx) {
    Room m;
    size_t at = 0;
    const int depth = dx ? w.N : w.K, slab = slab_columns(w, dx);
    m.x.base = (uint16_t*) base;
    m.x.rows = rows; m.x.cols = depth; m.x.ld = plane::padded(depth); m.x.batches = 1;
    at += plane::plane_bytes(Terms<T>::X, 1, rows, depth);
    m.w.base = (uint16_t*) (base + at);
    m.w.rows = dx ? w.N : slab; m.w.cols = dx ? slab : w.K; m.w.ld = plane::padded(m.w.cols); m.w.batches = 1;
    const size_t planes_end = at + plane::plane_bytes(Terms<T>::W, 1, m.w.rows, m.w.cols);
    // Where tiles are never cut (option "k_pieces" 1) nothing is ever stored in the parts' room, and planes of w that x has no like of
    // lie in it: workspaces of one plane are large enough then.
    m.cut = option_get(OPT_K_PIECES) != 1;
    at += plane::plane_bytes(m.cut ? Terms<T>::W : std::min(Terms<T>::X, Terms<T>::W), 1, m.w.rows, m.w.cols);
    m.parts = (float*) (base + at);
    const long long blocks = (depth + plane::BK - 1) / plane::BK;
    at += std::max(plane::parts_bytes(plane::count_tiles(rows, slab, 1, false, 128) * blocks, false),
                   plane::parts_bytes(plane::count_tiles(rows, slab, 1, false, 256) * blocks, true));
    m.bytes = std::max(at, planes_end);
    return m;
}

template <typename T>
int run(const Q4View& w, const void* in, long long ld_in, const void* bias, void* out, long long ld_out, int rows, bool dx, void* workspace,
        DeviceState* st, cudaStream_t s) {
    using K = Terms<T>;
    Room m = lay_out<T>((char*) workspace, w, rows, dx);
    int* launches = &thread_stats()->launches;
    int rc;
    const int depth = dx ? w.N : w.K, cols = dx ? w.K : w.N, slab = slab_columns(w, dx);
    const bool aligned = (uintptr_t) in % 16 == 0 && ld_in * (long long) sizeof(T) % 16 == 0;
    if (sizeof(T) == 2 && K::X == 1 && aligned && ld_in < (1LL << 31)) {  // BF16 rows that TMA can read where they lie
        m.x.base = (uint16_t*) in;
        m.x.ld = (int) ld_in;
    } else {
        const long long threads = (long long) rows * ((depth + 7) / 8);
        split_rows_kernel<T, K::X><<<(unsigned) ((threads + 255) / 256), 256, 0, s>>>((const T*) in, ld_in, rows, depth, aligned, m.x);
        CAKE_CUDA_OK(cudaGetLastError());
        *launches += 1;
    }
    plane::OperandMaps map_x, map_w;
    if ((rc = plane::encode_planes<Bf16Planes>(map_x.m, m.x, K::X))) return rc;
    for (int c0 = 0; c0 < cols; c0 += slab) {
        const int n = std::min(slab, cols - c0);
        Planes p = m.w;
        (dx ? p.cols : p.rows) = n;
        p.ld = plane::padded(p.cols);
        const int rt0 = dx ? 0 : c0 / 16, rts = (p.rows + 15) / 16, kb0 = dx ? c0 / 64 : 0, kbs = (p.cols + 63) / 64;
        expand_kernel<K::W><<<(unsigned) (((long long) rts * kbs * 32 + 255) / 256), 256, 0, s>>>(w, rt0, rts, kb0, kbs, p);
        CAKE_CUDA_OK(cudaGetLastError());
        *launches += 1;
        if ((rc = plane::encode_planes<Bf16Planes>(map_w.m, p, K::W))) return rc;
        typename RowsEpilogue<T>::Args ep;
        ep.out = (T*) out + c0;
        ep.ld = ld_out;
        ep.rows = rows;
        ep.cols = n;
        ep.bias = bias ? (const T*) bias + c0 : nullptr;
        ep.vec = (uintptr_t) ep.out % 16 == 0 && ld_out * (long long) sizeof(T) % 16 == 0;
        plane::Problem problem = {};
        problem.batch = 1;
        problem.a_turn = plane::ALONG;
        problem.b_turn = dx ? plane::DOWN : plane::ALONG;
        problem.chunk = K::CHUNK;
        problem.parts = m.cut ? m.parts : nullptr;
        problem.status_word = st->status_word;
        if ((rc = plane::launch<Bf16Planes, K::X, K::W, K::PRODUCTS, RowsEpilogue<T>>(map_x, map_w, problem, rows, n, depth, ep, st->sm_count, s, launches)))
            return rc;
    }
    return CAKEB200_OK;
}

}  // namespace

size_t q4_gemm_workspace(const Q4View& w, int rows, int type, bool dx) {
    return type == CAKEB200_F32 ? lay_out<float>(nullptr, w, rows, dx).bytes
           : type == CAKEB200_F16 ? lay_out<__half>(nullptr, w, rows, dx).bytes : lay_out<__nv_bfloat16>(nullptr, w, rows, dx).bytes;
}

int launch_q4_gemm(const Q4View& w, const void* in, long long ld_in, const void* bias, void* out, long long ld_out, int rows, int type, bool dx,
                   void* workspace, DeviceState* st, cudaStream_t s) {
    if (type == CAKEB200_F32) return run<float>(w, in, ld_in, bias, out, ld_out, rows, dx, workspace, st, s);
    if (type == CAKEB200_F16) return run<__half>(w, in, ld_in, bias, out, ld_out, rows, dx, workspace, st, s);
    return run<__nv_bfloat16>(w, in, ld_in, bias, out, ld_out, rows, dx, workspace, st, s);
}

}  // namespace cakeb200
