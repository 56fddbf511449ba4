// Block-scaled fp8 products: argument checks, plan and entry points (kernels: gemm_block_tile.hip, gemm_block_rows.hip).
#include <algorithm>
#include <cmath>

#include "gemm_block.h"

namespace llmq {
namespace {

// cfg: a tile configuration, or kRowsCfg + a variant of the row-streaming kernel
struct BlockPlan { int cfg, splits, blocks_per_split; };
constexpr int kRowsCfg = kNumBlockTiles;
thread_local int forced_cfg = -1, forced_splits = 0;

// What a launch takes, in us, as a rule of the sizes alone:
//   start + max(stream, loop) + 0.15 min(stream, loop) + what a K split adds
// stream: the operands once at 6.6 TB/s, longer where some CUs have a block more than others.  loop: steps along K times what one takes, from
// `alone` (a few blocks on the chip) to `alone` + `crowd` (one on every CU); with more blocks than CUs `full` for each of a CU's, and `turn` from one to the next
// (outputs out, first operands in); a last round that is not full costs as the fourth root of what it holds (row-streaming kernel: all of it).  A split
// adds a launch and its sums' way out and back.
// Fitted to random sizes (1-8192 tokens, 128-37888 channels, K 512-18944; up to 128 experts), every configuration and split timed with the weights out of
// HBM.  The choice is slower than the fastest of the size by, on average and in the worst 5 % of the sizes: 1.4 % and 9 % (3900 sizes of more than 64
// tokens), 2.0 % and 12 % (2000 of fewer), 1.9 % and 10 % (4000 by experts).  Without `turn` it was 1.8, 2.2 and 2.7 % on average.
struct Cost { float start, alone, full, crowd, turn; };
constexpr Cost kTileCost[kNumBlockTiles] = {{7.27, 1.27, 1.86, 0.544, 8.63}, {5.63, 0.639, 1.05, 0.417, 4.86}, {5.37, 0.325, 0.676, 0.411, 2.65}, {4.55, 0.363, 0.405, 0.124, 0.823},
                                            {3.75, 0.319, 0.313, 0.043, 0.559}, {4.05, 0.281, 0.286, 0.049, 0.621}, {5.4, 0.466, 0.792, 0.29, 2.17}, {4.76, 0.344, 0.575, 0.182, 2.49}};
constexpr Cost kRowsCost[kNumBlockRows] = {{2.74, 0.343, 0.298, 0.025, 0.417}, {3.04, 0.55, 0.655, 0.119, 1.52}, {2.9, 0.402, 0.356, 0.057, 0.402}, {3.07, 0.532, 0.605, 0.057, 1.59},
                                           {3.28, 0.706, 0.714, 0.116, 2.61}, {3.18, 0.646, 0.794, 0.092, 1.39}, {3.34, 0.56, 0.888, 0.545, 0.384}};

float cost_us(const Cost& c, double blocks, double steps, double bytes, bool rows) {
    const float r = (float)(blocks / 256.0), whole = floorf(r), rest = r - whole;
    const float step = c.alone + c.crowd * std::min(r, 1.f);
    float rounds = 1.f, stream = (float)(bytes / 6.6e6);
    if (r > 1.f) {
        rounds = whole + (rows ? ceilf(rest) : sqrtf(sqrtf(rest)));
        stream *= 1.f + 0.3f * (ceilf(r) / r - 1.f);
    }
    const float loop = std::max((float)steps * step, rounds > 1.f ? (float)steps * c.full * rounds + c.turn * (rounds - 1.f) : 0.f);
    return c.start + std::max(stream, loop) + 0.15f * std::min(stream, loop);
}

BlockPlan search(int64_t M, int64_t N, int64_t K) {
    const int KB = (int)((K + kScaleBlock - 1) / kScaleBlock);
    BlockPlan best = {0, 1, KB};
    float least = 3e38f;
    for (int c = 0; c < kNumBlockTiles; c++) {
        const BlockTile& t = kBlockTiles[c];
        const double tiles = (double)((M + t.bm - 1) / t.bm) * (double)((N + t.bn - 1) / t.bn);
        for (int s : {1, 2, 3, 4, 6, 8}) {
            if (s > 1 && (KB / s < 4 || tiles * s > (t.bm * t.bn > 64 * 128 ? 300 : 600))) break;
            const int per = (KB + s - 1) / s, splits = (KB + per - 1) / per;
            float us = cost_us(kTileCost[c], tiles * splits, (per + t.ks - 1) / t.ks, (double)N * K + (double)M * K, false);
            if (splits > 1) us += 3.f + (float)(splits * (double)M * N * 8 / 7e6);
            if (us < least) least = us, best = {c, splits, per};
        }
    }
    for (int v = 0; v < kNumBlockRows; v++) {
        const BlockRows& r = kBlockRows[v];
        if (M > 16 * r.mt) continue;
        const float us = cost_us(kRowsCost[v], (double)((N + 16 * r.t - 1) / (16 * r.t)), (KB + 4 * r.steps - 1) / (4 * r.steps), (double)N * K, true);
        if (us < least) least = us, best = {kRowsCfg + v, 1, KB};
    }
    return best;
}

BlockPlan plan(int64_t M, int64_t N, int64_t K) {
    const int KB = (int)((K + kScaleBlock - 1) / kScaleBlock);
    if (forced_cfg >= kRowsCfg && M <= 16 * kBlockRows[forced_cfg - kRowsCfg].mt) return {forced_cfg, 1, KB};
    if (forced_cfg >= 0 && forced_cfg < kRowsCfg) {
        const int want = std::max(1, std::min({forced_splits, KB, kMostSplits})), per = (KB + want - 1) / want;
        return {forced_cfg, (KB + per - 1) / per, per};
    }
    thread_local int64_t of[3] = {0, 0, 0};  // the last size
    thread_local BlockPlan last;
    if (of[0] != M || of[1] != N || of[2] != K) last = search(M, N, K), of[0] = M, of[1] = N, of[2] = K;
    return last;
}

// The host knows the rows of all experts together, not each one's: every expert that may have rows is taken to end with about half a tile.
int plan_grouped(int64_t rows, int64_t experts, int64_t N, int64_t K) {
    if (forced_cfg >= 0 && forced_cfg < kRowsCfg) return forced_cfg;
    thread_local int64_t of[4] = {0, 0, 0, 0};
    thread_local int last;
    if (of[0] == rows && of[1] == experts && of[2] == N && of[3] == K) return last;
    const int KB = (int)((K + kScaleBlock - 1) / kScaleBlock);
    const double used = (double)std::min(rows, experts);
    float least = 3e38f;
    for (int c = 0; c < kNumBlockTiles; c++) {
        const BlockTile& t = kBlockTiles[c];
        const double tiles = std::max(used, (double)rows / t.bm + 0.45 * used) * (double)((N + t.bn - 1) / t.bn);
        const float us = cost_us(kTileCost[c], tiles, (KB + t.ks - 1) / t.ks, used * (double)N * K + (double)rows * K, false);
        if (us < least) least = us, last = c;
    }
    of[0] = rows, of[1] = experts, of[2] = N, of[3] = K;
    return last;
}

size_t partial_bytes(const BlockPlan& p, int64_t M, int64_t N) { return p.splits > 1 ? (size_t)p.splits * (size_t)M * (size_t)partial_ld(N) * 4 : 0; }

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
    return launch_block_tile(plan_grouped(M, experts, N, K), 1, g, (hipStream_t)stream);
}

extern "C" int llmq_gemm_fp8_block_force_plan(int cfg, int splits) {
    if (cfg >= kNumBlockTiles + kNumBlockRows || splits < 0) return LLMQ_ERR_SHAPE;
    forced_cfg = cfg < 0 ? -1 : cfg;
    forced_splits = splits;
    return LLMQ_OK;
}
