// What the two files of 8-bit products share.
#pragma once
#include "blocks8.h"

constexpr int kTileRowBlocks = 4;    // packed blocks of 64 rows of w a tile

struct BlocksCall {
    bf16_t* out;                     // [M][ldo], or null: the float32 sums are the result
    unsigned char* rows8;            // or silu(gate) * up in 8 bits: codes [M][128 ceil(N / 256)] and their scales [ceil(N / 256)][scale_stride]
    unsigned char* rows8_scales;
    const unsigned char* a;          // codes [M][128 blocks]
    const unsigned char* a_scales;   // [blocks][scale_stride]
    const bf16_t* rows;              // or rows of 128 blocks values, lda apart, that the few-row kernels bring to 8 bits
    size_t lda;
    const unsigned char* wp;         // packed codes of N rows
    const unsigned char* w_scales;   // [N / 64][blocks][4]
    const float* bias;
    float* sums;                     // [parts][M][64 ceil(N / 64)] of a product in parts of k; [M][N] of the few-row kernels without out
    size_t scale_stride;
    int M, N, blocks, ldo;
    bool once;                       // wp will not be in the last-level cache when it is read next
};

__device__ __forceinline__ i32x8_8 two_pieces(u32x4_8 a, u32x4_8 b) {
    i32x8_8 v;
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = (int)a[e], v[4 + e] = (int)b[e];
    return v;
}

// (of many rows, gemm_blocks_tiles.hip; n_full: row tiles in tiles of 16 token_tiles tokens, 0: all)
int launch_blocks_tiles(const BlocksCall& c, bool gated, int token_tiles, int groups, int n_full, int parts, hipStream_t stream);
