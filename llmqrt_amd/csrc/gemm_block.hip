// Block-scaled fp8 products: argument checks, plan and entry points (kernels: gemm_block_tile.hip, gemm_block_rows.hip).
#include <algorithm>

#include "gemm_block.h"

namespace llmq {
namespace {

struct BlockPlan { int cfg, splits, blocks_per_split; };
thread_local int forced_cfg = -1, forced_splits = 0;

BlockPlan split_plan(int cfg, int splits, int KB) {
    const int per = (KB + splits - 1) / splits;
    return {cfg, (KB + per - 1) / per, per};
}

// cfg: a tile configuration, or kRowsCfg + a variant of the row-streaming kernel
constexpr int kRowsCfg = kNumBlockTiles;
bool rows_take(int cfg, int64_t M) { return M <= 16 * kBlockRows[cfg - kRowsCfg].mt; }

BlockPlan plan(int64_t M, int64_t N, int64_t K) {
    const int KB = (int)((K + kScaleBlock - 1) / kScaleBlock);
    if (forced_cfg >= 0 && (forced_cfg < kRowsCfg || rows_take(forced_cfg, M)))
        return forced_cfg >= kRowsCfg ? BlockPlan{forced_cfg, 1, KB} : split_plan(forced_cfg, std::max(1, std::min(forced_splits, KB)), KB);
    if (M <= 16) return {kRowsCfg + (N > 8192 ? 8 : 0), 1, KB};
    if (M <= 32) return {kRowsCfg + (N > 8192 ? 5 : 3), 1, KB};
    if (M <= 48) return {kRowsCfg + (N > 8192 ? 11 : 10), 1, KB};
    if (M <= 64) return {kRowsCfg + (N > 8192 ? 7 : 6), 1, KB};
    const int cfg = M <= 32 ? 4 : M <= 64 ? 3 : M <= 1024 ? 2 : 0;
    const BlockTile t = kBlockTiles[cfg];
    const int64_t tiles = ((M + t.bm - 1) / t.bm) * ((N + t.bn - 1) / t.bn);
    const int splits = (int)std::max<int64_t>(1, std::min<int64_t>(256 / tiles, KB / 8));
    return split_plan(cfg, splits, KB);
}

int plan_grouped(int64_t rows, int64_t experts) {
    if (forced_cfg >= 0 && forced_cfg < kRowsCfg) return forced_cfg;
    const int64_t each = rows / experts;
    return each <= 32 ? 4 : each <= 64 ? 3 : each <= 256 ? 2 : 0;
}

size_t partial_bytes(const BlockPlan& p, int64_t M, int64_t N) { return p.splits > 1 ? (size_t)p.splits * (size_t)M * (size_t)N * 4 : 0; }

constexpr int64_t kMaxLd = 1 << 23;  // 256 rows stay within 32-bit offsets

int check(const uint8_t* A, int64_t lda, const float* sa, const uint8_t* B, int64_t ldb, const float* sw, const void* bias, int bias_dtype,
          const void* out, int out_dtype, int64_t ldo, int64_t M, int64_t N, int64_t K) {
    if (out_dtype != LLMQ_BF16 && out_dtype != LLMQ_F16) return LLMQ_ERR_DTYPE;
    if (bias && bias_dtype != LLMQ_BF16 && bias_dtype != LLMQ_F16 && bias_dtype != LLMQ_F32) return LLMQ_ERR_DTYPE;
    if (M < 0 || N < 0 || K < 0 || M > 0x7fffff00LL || N > 0x7fffff00LL || K % 16 || lda < K || ldb < K || lda % 16 || ldb % 16 || lda > kMaxLd ||
        ldb > kMaxLd || ldo < N)
        return LLMQ_ERR_SHAPE;
    if (M == 0 || N == 0) return LLMQ_OK;
    if (K == 0) return LLMQ_ERR_SHAPE;
    if (!A || !sa || !B || !sw || !out) return LLMQ_ERR_NULL;
    if (!aligned16(A) || !aligned16(B)) return LLMQ_ERR_ALIGN;
    return LLMQ_OK;
}

}  // namespace
}  // namespace llmq

using namespace llmq;

extern "C" size_t llmq_gemm_fp8_block_workspace_bytes(int64_t M, int64_t N, int64_t K) {
    if (M <= 0 || N <= 0 || K <= 0 || M > 0x7fffff00LL || N > 0x7fffff00LL || K > kMaxLd) return 0;
    return partial_bytes(plan(M, N, K), M, N);
}

extern "C" int llmq_gemm_fp8_block(const uint8_t* A, int64_t lda, const float* a_scale, const uint8_t* B, int64_t ldb, const float* w_scale,
                                   const void* bias, int bias_dtype, void* out, int out_dtype, int64_t ldo, int64_t M, int64_t N, int64_t K,
                                   void* workspace, size_t workspace_bytes, llmq_stream_t stream) {
    const int rc = check(A, lda, a_scale, B, ldb, w_scale, bias, bias_dtype, out, out_dtype, ldo, M, N, K);
    if (rc != LLMQ_OK || M == 0 || N == 0) return rc;
    const BlockPlan p = plan(M, N, K);
    const size_t need = partial_bytes(p, M, N);
    if (need && (!workspace || workspace_bytes < need)) return LLMQ_ERR_WORKSPACE;
    if (need && !aligned16(workspace)) return LLMQ_ERR_ALIGN;
    BlockArgs g = {};
    g.A = A, g.sa = a_scale, g.B = B, g.sw = w_scale, g.bias = bias, g.out = out, g.partials = (float*)workspace;
    g.lda = lda, g.ldb = ldb, g.ldo = ldo, g.M = (int)M, g.N = (int)N, g.K = (int)K;
    g.KB = (int)((K + kScaleBlock - 1) / kScaleBlock), g.NB = (int)((N + kScaleBlock - 1) / kScaleBlock), g.experts = 1;
    g.blocks_per_split = p.blocks_per_split, g.bias_dtype = bias_dtype, g.out_dtype = out_dtype;
    if (p.cfg >= kRowsCfg) return launch_block_rows(p.cfg - kRowsCfg, g, (hipStream_t)stream);
    return launch_block_tile(p.cfg, p.splits, g, (hipStream_t)stream);
}

extern "C" int llmq_gemm_fp8_block_grouped(const uint8_t* A, int64_t lda, const float* a_scale, const uint8_t* B, const float* w_scale,
                                           const int32_t* offsets, int64_t experts, const void* bias, int bias_dtype, void* out, int out_dtype,
                                           int64_t ldo, int64_t M, int64_t N, int64_t K, llmq_stream_t stream) {
    if (experts < 0 || experts > 65536) return LLMQ_ERR_SHAPE;
    const int rc = check(A, lda, a_scale, B, K, w_scale, bias, bias_dtype, out, out_dtype, ldo, M, N, K);
    if (rc != LLMQ_OK || M == 0 || N == 0 || experts == 0) return rc;
    if (!offsets) return LLMQ_ERR_NULL;
    BlockArgs g = {};
    g.A = A, g.sa = a_scale, g.B = B, g.sw = w_scale, g.bias = bias, g.out = out, g.offsets = offsets;
    g.lda = lda, g.ldb = K, g.ldo = ldo, g.M = (int)M, g.N = (int)N, g.K = (int)K;
    g.KB = (int)((K + kScaleBlock - 1) / kScaleBlock), g.NB = (int)((N + kScaleBlock - 1) / kScaleBlock), g.experts = (int)experts;
    g.bias_dtype = bias_dtype, g.out_dtype = out_dtype;
    return launch_block_tile(plan_grouped(M, experts), 1, g, (hipStream_t)stream);
}

extern "C" int llmq_gemm_fp8_block_force_plan(int cfg, int splits) {
    if (cfg >= kNumBlockTiles + kNumBlockRows || splits < 0) return LLMQ_ERR_SHAPE;
    forced_cfg = cfg < 0 ? -1 : cfg;
    forced_splits = splits;
    return LLMQ_OK;
}
