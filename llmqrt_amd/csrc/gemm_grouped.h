// W8A8 product by experts: what the tile kernel (gemm_tile_i8_grouped.hip, also the planner and entry point) and the row-streaming kernel
// (gemm_rows_i8_grouped.hip) share.
#pragma once
#include "gemm_tile.h"
#include "llmq_common.h"

namespace llmq {

struct GroupedCall {
    const uint8_t *A, *B;    // int8 [M, K], [experts, N, K]
    int64_t lda, ldo;
    int M, N, K;
    Epilogue ep;             // scales, bias; of expert 0
    void* out;
    const int32_t* offsets;  // experts + 1
    int experts;
};

// Variants of the row-streaming kernel: 16-channel and 16-row tiles of a block, LDS stages, blocks that a CU holds.  At most so many experts.
// (4 x 16 channels, and 32 or 64 rows: each ahead of these two in some sizes, none by enough to matter: the best of all 0.3 % under the best of the ones kept, on average.)
#define LLMQ_GROUPED_ROWS(V) V(0, 1, 1, 4, 2) V(1, 2, 1, 3, 2)
struct GroupedRows { int t, mt, per_cu; };
constexpr GroupedRows kGroupedRows[] = {
#define LLMQ_GROUPED_ROWS_SHAPE(I, T, MT, NS, CU) {T, MT, CU},
    LLMQ_GROUPED_ROWS(LLMQ_GROUPED_ROWS_SHAPE)
#undef LLMQ_GROUPED_ROWS_SHAPE
};
constexpr int kNumGroupedRows = sizeof(kGroupedRows) / sizeof(kGroupedRows[0]), kGroupedRowsExperts = 512;

int launch_grouped_rows(int variant, const GroupedCall& g, hipStream_t st);

}  // namespace llmq
