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
// Scales (16 bit) and zero points (8 bit) follow, 16 per block row and group, the ones of rows a and a + 8 adjacent.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace cakeb200 {

struct Q4View {
    const uint4* codes;       // [row_tiles][k_blocks][32 lanes]
    const uint16_t* scales;   // [row_tiles][groups][16]
    const uint8_t* zeros;     // same, or nullptr
    int N, K;                 // out_features, in_features
    int group, groups;        // groups: of the features padded to whole blocks
    int row_tiles, k_blocks;
    int scale_bf16;
};

inline __host__ __device__ int q4_row_tiles(int N) { return (N + 15) / 16; }
inline __host__ __device__ int q4_k_blocks(int K) { return (K + 63) / 64; }
inline __host__ __device__ int q4_groups(int K, int group) { return (q4_k_blocks(K) * 64 + group - 1) / group; }
// place of local row i (0..15) of a block row among its 16 scales
inline __host__ __device__ int q4_scale_place(int i) { return (i & 7) * 2 + (i >> 3); }

// Checks the descriptor (no device access) and fills the view.
int q4_view(const cakeb200_q4* w, const char* who, Q4View* out);

#ifdef __CUDACC__
__device__ __forceinline__ float q4_scale(uint16_t bits, int is_bf16) {
    return is_bf16 ? __uint_as_float((uint32_t) bits << 16) : __half2float(__ushort_as_half(bits));
}
#endif

}  // namespace cakeb200
