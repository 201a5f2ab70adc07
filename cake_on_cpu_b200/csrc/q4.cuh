// Weights held in 4 bits: the packed form shared by the kernels that read it.
//
//   w[n, k] = s[n, g] * (q[n, k] - z[n, g]),   g = k / group,   q in 0..15,   z = 8 where no zero points are given.
//
// The packed form is the fragment order of mma.m16n8k16 with the weights as the A operand, so that one 16-byte
// load per lane brings a warp a block of 16 output features x 64 input features and nothing has to be exchanged
// between lanes.  Lane 4 a + t of a block (a = 0..7, t = 0..3) holds rows a and a + 8; its word j = 0..3 holds the
// eight codes of MMA j, which covers the input features
//     k = 32 (j / 2) + 8 t + 4 (j & 1) + {0, 1, 2, 3},    t = 0..3,
// i.e. words 0 and 1 lie in the block's first 32 features and words 2 and 3 in the other 32 (the smallest group), and a
// lane's features of a word pair are eight consecutive ones (one 16-byte load of a 16-bit x).  In a word,
//     bits [4 i, 4 i + 4) and [16 + 4 i, 16 + 4 i + 4),   i = 0..3,
// hold the pair of consecutive features (k, k + 1) of fragment register i: i & 1 picks row a or a + 8, i >> 1 the
// lower or upper pair.  A mask and a shift then leave a pair of codes in the two halves of a register.
//
// Blocks come in pairs, 128 features (a "step", the largest group).  Scales (16 bit) and then zero points (8 bit) follow the
// codes, for every block row and step those of rows a and a + 8 of its 1, 2 or 4 groups: [a][group][row a, row a + 8], one load
// per lane.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace cakeb200 {

struct Q4View {
    const uint4* codes;       // [row_tiles][2 steps][32 lanes]
    const uint16_t* scales;   // [row_tiles][steps][8][groups of a step][2]
    const uint8_t* zeros;     // same, or nullptr
    int N, K;                 // out_features, in_features
    int group_shift;          // the group is 1 << group_shift features
    int row_tiles, steps;
    int scale_bf16;
};

inline __host__ __device__ int q4_row_tiles(int N) { return (N + 31) / 32 * 2; }  // in pairs, as the forward product takes them
inline __host__ __device__ int q4_steps(int K) { return (K + 127) / 128; }
// Place of the scale of local row i (0..15) of a block row for the group that holds feature k of its step (0..127).
inline __host__ __device__ int q4_scale_place(int i, int k, int group_shift) {
    return (((i & 7) << (7 - group_shift)) + (k >> group_shift)) * 2 + (i >> 3);
}
// Scales of a block row and step: 16 for each of its groups.
inline __host__ __device__ long long q4_scale_at(const Q4View& w, int rt, int step) {
    return ((long long) rt * w.steps + step) << (4 + 7 - w.group_shift);
}

// Checks the descriptor (no device access) and fills the view.
int q4_view(const cakeb200_q4* w, const char* who, Q4View* out);

// Products with many rows (q4_gemm.cu); type: CAKEB200_F32, _F16 or _BF16.
size_t q4_gemm_workspace(const Q4View& w, int rows, int type, bool dx);
int launch_q4_gemm(const Q4View& w, const void* in, long long ld_in, const void* bias, void* out, long long ld_out, int rows, int type, bool dx,
                   void* workspace, DeviceState* st, cudaStream_t s);

#ifdef __CUDACC__
__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ float from_float<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// v = t0 + t1 + ... with every term a bf16 (the upper half of an FP32), by truncation; a pair of values at a time.
// Terms of a value that is not finite are not all finite.
template <int TERMS>
__device__ __forceinline__ void split_pair(float v0, float v1, uint32_t* out) {
#pragma unroll
    for (int t = 0; t < TERMS; t++) {
        out[t] = __byte_perm(__float_as_uint(v0), __float_as_uint(v1), 0x7632);
        if (t + 1 < TERMS) {
            v0 -= __uint_as_float(__float_as_uint(v0) & 0xffff0000u);
            v1 -= __uint_as_float(__float_as_uint(v1) & 0xffff0000u);
        }
    }
}

// The same in two terms, each rounded to nearest: within 2^-17 of v, on either side of it.
__device__ __forceinline__ void round_pair(float v0, float v1, uint32_t* out) {
#pragma unroll
    for (int t = 0; t < 2; t++) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(v0, v1);
        out[t] = *reinterpret_cast<const uint32_t*>(&h);
        v0 -= __uint_as_float(out[t] << 16);
        v1 -= __uint_as_float(out[t] & 0xffff0000u);
    }
}

__device__ __forceinline__ float q4_scale(uint16_t bits, int is_bf16) {
    return is_bf16 ? __uint_as_float((uint32_t) bits << 16) : __half2float(__ushort_as_half(bits));
}
#endif

}  // namespace cakeb200
