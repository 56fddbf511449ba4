// Block-scaled fp8 products (one scale per token and 128 of K, one per 128 x 128 weights), alone and by experts: what the kernels
// (gemm_block_tile.hip) and the planner and entry points (gemm_block.hip) share.
#pragma once
#include "llmq_common.h"

namespace llmq {

constexpr int kScaleBlock = 128;
constexpr int kMostSplits = 8;  // of K

__host__ __device__ inline int64_t partial_ld(int64_t N) { return (N + 7) & ~(int64_t)7; }

struct BlockArgs {
    const uint8_t* A;      // [M, K] e4m3
    const float* sa;       // [M, KB]
    const uint8_t* B;      // [N, K] e4m3, of expert 0
    const float* sw;       // [NB, KB], of expert 0
    const void* bias;      // [N] of expert 0, or null
    void* out;             // [M, N]
    const int32_t* offsets;  // experts + 1 first rows, or null: one matrix for all rows
    float* partials;       // K split: [splits, M, partial_ld(N)]
    int64_t lda, ldb, ldo;
    int M, N, K, KB, NB, experts;
    int blocks_per_split;  // of 128 of K
    int bias_dtype, out_dtype;
};

struct BlockTile { int bm, bn, ks; };  // tokens, channels, groups of wavefronts of a block
constexpr BlockTile kBlockTiles[] = {
    {256, 256, 1},  // 0: 8 wavefronts of 128 x 64
    {128, 256, 1},  // 1: 8 wavefronts of 64 x 64
    {64, 256, 1},  // 2: 8 wavefronts of 32 x 64
    {64, 128, 1},  // 3: 4 wavefronts of 32 x 64
    {32, 128, 1},  // 4: 4 wavefronts of 32 x 32
    {64, 64, 1},  // 5: 4 wavefronts of 32 x 32
    {64, 128, 2},  // 6: 2 groups of 4 wavefronts of 32 x 64
    {64, 64, 2},  // 7: 2 groups of 4 wavefronts of 32 x 32
};
constexpr int kNumBlockTiles = sizeof(kBlockTiles) / sizeof(kBlockTiles[0]);

// Variants of gemm_block_rows.hip: 16-channel and 16-token tiles of a block, blocks of K per wavefront and stage, stages; several groups of channels
// per block.  They take up to 16 MT tokens.
#define LLMQ_BLOCK_ROWS(V)                                                                              \
    V(0, 1, 1, 1, 4, false) V(1, 1, 1, 2, 4, false) V(2, 1, 2, 1, 3, false) V(3, 1, 3, 1, 4, false)      \
    V(4, 2, 3, 1, 3, false) V(5, 1, 4, 1, 3, false) V(6, 4, 1, 1, 3, true)
struct BlockRows { int t, mt, steps; };
constexpr BlockRows kBlockRows[] = {
#define LLMQ_BLOCK_ROWS_SHAPE(I, T, MT, STEPS, NS, MANY) {T, MT, STEPS},
    LLMQ_BLOCK_ROWS(LLMQ_BLOCK_ROWS_SHAPE)
#undef LLMQ_BLOCK_ROWS_SHAPE
};
constexpr int kNumBlockRows = sizeof(kBlockRows) / sizeof(kBlockRows[0]);

int launch_block_rows(int variant, const BlockArgs& g, hipStream_t st);
int launch_block_tile(int cfg, int splits, const BlockArgs& g, hipStream_t st);

}  // namespace llmq
