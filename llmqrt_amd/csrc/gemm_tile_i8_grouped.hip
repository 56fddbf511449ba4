// W8A8 product by experts: the int8 tile kernel of gemm_tile_impl.h over rows that are sorted by expert.
//
//   out[m, n] = dtype( (acc[m, n] a_scale[m]) w_scale[e, n] + bias[e, n] ),  acc[m, n] = sum_k A[m, k] B[e, n, k],  m of expert e
//
// The host does not know the experts' rows, so the grid is what any distribution can need (each expert may end with a tile that is not full) and a block
// finds its tile from the offsets.
//
// Bound by the matrix cores (and the power that they take) where experts have many rows, by the weights out of HBM where they have few.  Tiles of 256 x 256, 128 x 256,
// 256 x 128, 192 x 128, 128 x 128, us: 32768 rows of 32 experts, 4864 x 3584, 595 (1.92 POP/s; one matrix of that size 592) 660 664 709 821; 1998 rows of 16, 3584 x 1536, 26
// 37 32 31 36; 12151 rows of 5, 293 x 800, 19.6 13.4 13.4 11.5 16.2.  32 x 128 and 64 x 128 are for a few rows each (gemm_rows_i8_grouped.hip).
#include <cmath>

#include "expert_tiles.h"
#include "gemm_grouped.h"
#include "gemm_tile_impl.h"

namespace llmq {
namespace {

struct ManyMatrices {
    static constexpr bool GROUPED = true;
    const int32_t* offsets;  // experts + 1
    int experts;
    template <int BM>
    __device__ __forceinline__ bool tile(int M, int tiles_n, int& expert, int& row0, int& row_end, int& tn) const {
        return expert_tile<BM>(offsets, experts, M, tiles_n, expert, row0, row_end, tn);
    }
};

template <class C>
int launch_grouped(const GroupedCall& g, hipStream_t st) {
    const bool kfull = g.K % C::BK == 0;
    const auto kernel = kfull ? gemm_tile_kernel<C, true, ManyMatrices> : gemm_tile_kernel<C, false, ManyMatrices>;
    if (C::LDS_BYTES > 65536u) {
        static bool raised[2][64] = {};  // per device: the attribute belongs to the loaded code object of the current device
        int dev = 0;
        if (hipGetDevice(&dev) != hipSuccess) return LLMQ_ERR_LAUNCH;
        if (dev < 0 || dev >= 64 || !raised[kfull][dev]) {
            if (hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)C::LDS_BYTES) != hipSuccess)
                return LLMQ_ERR_LAUNCH;
            if (dev >= 0 && dev < 64) raised[kfull][dev] = true;  // benign if two threads race here: both set the same value
        }
    }
    const int64_t tiles_n = cdiv(g.N, C::BN), tiles_m = g.M / C::BM + std::min(g.experts, g.M);
    if (tiles_m * tiles_n * C::NT > 0xffffffffLL) return LLMQ_ERR_SHAPE;  // threads of a grid
    hipLaunchKernelGGL(kernel, dim3((unsigned)(tiles_m * tiles_n)), dim3(C::NT), C::LDS_BYTES, st, g.A, g.lda, g.B, (int64_t)g.K, g.M, g.N, g.K, g.K, g.ep,
                       g.out, g.ldo, (void*)nullptr, (void*)nullptr, ManyMatrices{g.offsets, g.experts});
    return launch_status();
}

thread_local int forced = -1;  // llmq_gemm_w8a8_grouped_force_plan

// What a launch takes, in us, as a rule of the sizes alone; the host knows the rows of all experts together, not each one's, and takes every expert that may
// have rows to end with about half a tile:
//   start + max(stream, loop) + 0.15 min(stream, loop)
// stream: the operands once at `rate` TB/s.  loop: steps along K (128 bytes, 512 of the row-streaming kernel) times what one takes, from `alone` (a few blocks on the
// chip) to `alone` + `crowd` (as many as it holds); with more, `full` for each of a CU's, and `turn` from one to the next; a last round of tiles that is not full
// costs as the fourth root of what it holds.
// Fitted to 4000 random sizes (1-32768 rows, 1-128 experts, 256-4864 channels, K 512-18944, unevenly used experts), every configuration timed with the weights out
// of HBM: the choice is slower than the size's fastest by 1.6 % on average and 10 % in the worst 5 % of the sizes.  Without the row-streaming kernel it would be 12 %.
struct Cost { double start, alone, full, crowd, turn, rate; };
constexpr int kFirstTile = 4, kNumTiles = kNumShapes - kFirstTile;
constexpr Cost kTileCost[kNumTiles] = {{4.48, 0.268, 0.429, 0.158, 3.35, 5.81}, {2.92, 0.231, 0.572, 0.118, 1.29, 6.2}, {15.1, 0.691, 2.04, 0.652, 8.32, 33.9},
                                       {10, 0.492, 1.26, 0.511, 7.81, 11.3},    {5.41, 0.384, 0.872, 0.227, 5.34, 12.3}, {6.98, 0.477, 0.992, 0.309, 7, 22.5},
                                       {9.08, 0.523, 1.23, 0.468, 7.02, 31.9}};
constexpr Cost kRowsCost[kNumGroupedRows] = {{1.94, 0.142, 0.769, 0.838, 0.993, 3.5}, {2.44, 0.446, 0.769, 0.372, 1.73, 11.2}};

int search(double M, double experts, double N, double K) {
    const double used = std::min(M, experts), bytes = (used * N * K + M * K) / 1e6;
    double least = 1e300;
    int best = kFirstTile;
    auto consider = [&](const Cost& c, int cfg, double loop) {
        const double stream = bytes / c.rate, us = c.start + std::max(stream, loop) + 0.15 * std::min(stream, loop);
        if (us < least) least = us, best = cfg;
    };
    for (int i = 0; i < kNumTiles; i++) {
        const Cost& c = kTileCost[i];
        const TileShape& t = kShapes[kFirstTile + i];
        const double r = std::max(used, M / t.bm + 0.45 * used) * std::ceil(N / t.bn) / kNumCu, steps = std::ceil(K / 128);
        double loop = steps * (c.alone + c.crowd * std::min(r, 1.0));
        if (r > 1) {
            const double whole = std::floor(r), rounds = whole + std::sqrt(std::sqrt(r - whole));
            loop = std::max(loop, steps * c.full * rounds + c.turn * (rounds - 1));
        }
        consider(c, kFirstTile + i, loop);
    }
    for (int i = 0; i < kNumGroupedRows && experts <= kGroupedRowsExperts; i++) {
        const Cost& c = kRowsCost[i];
        const GroupedRows& s = kGroupedRows[i];
        const double r = std::max(used, M / (16 * s.mt) + 0.45 * used) * std::ceil(N / (16 * s.t)) / kNumCu / s.per_cu, steps = std::ceil(K / 512);
        double loop = steps * (c.alone + c.crowd * std::min(r, 1.0));
        if (r > 1) loop = std::max(loop, (steps * c.full + c.turn) * r);
        consider(c, kNumShapes + i, loop);
    }
    return best;
}

int plan(int64_t M, int64_t experts, int64_t N, int64_t K) {
    thread_local int64_t of[4] = {0, 0, 0, 0};  // the last size
    thread_local int last;
    if (of[0] != M || of[1] != experts || of[2] != N || of[3] != K)
        last = search((double)M, (double)experts, (double)N, (double)K), of[0] = M, of[1] = experts, of[2] = N, of[3] = K;
    return last;
}

}  // namespace
}  // namespace llmq

using namespace llmq;

extern "C" int llmq_gemm_w8a8_grouped(const int8_t* A, int64_t lda, const float* a_scale, const int8_t* B, const float* w_scale, const int32_t* offsets,
                                      int64_t experts, const void* bias, int bias_dtype, void* out, int out_dtype, int64_t ldo, int64_t M, int64_t N,
                                      int64_t K, llmq_stream_t stream) {
    if (out_dtype != LLMQ_BF16 && out_dtype != LLMQ_F16) return LLMQ_ERR_DTYPE;
    if (bias && bias_dtype != LLMQ_BF16 && bias_dtype != LLMQ_F16 && bias_dtype != LLMQ_F32) return LLMQ_ERR_DTYPE;
    if (experts < 0 || experts > 65536 || M < 0 || N < 0 || K < 0 || M > 0x7fffff00LL || N > 0x7fffff00LL || K % 16 || K >= 1 << 17 || lda < K || lda % 16 ||
        lda > 1 << 23 || ldo < N)  // (131072 products of -128 and -128 leave the int32 range; 256 rows stay within 32-bit offsets)
        return LLMQ_ERR_SHAPE;
    if (M == 0 || N == 0 || experts == 0) return LLMQ_OK;
    if (K == 0) return LLMQ_ERR_SHAPE;
    if (!A || !a_scale || !B || !w_scale || !offsets || !out) return LLMQ_ERR_NULL;
    if (!aligned16(A) || !aligned16(B)) return LLMQ_ERR_ALIGN;
    GroupedCall g = {};
    g.A = (const uint8_t*)A, g.B = (const uint8_t*)B, g.lda = lda, g.ldo = ldo, g.M = (int)M, g.N = (int)N, g.K = (int)K, g.out = out;
    g.ep.a_scale = a_scale, g.ep.w_scale = w_scale, g.ep.bias = bias, g.ep.alpha = 1.f, g.ep.beta = 1.f;
    g.ep.bias_dtype = bias_dtype, g.ep.out_dtype = out_dtype;
    g.offsets = offsets, g.experts = (int)experts;
    const hipStream_t st = (hipStream_t)stream;
    const int cfg = forced >= 0 && (forced < kNumShapes || experts <= kGroupedRowsExperts) ? forced : plan(M, experts, N, K);
    if (cfg >= kNumShapes) return launch_grouped_rows(cfg - kNumShapes, g, st);
    switch (cfg) {
        case 4: return launch_grouped<GemmCfg<64, 128, 128, 2, 2, false, 0, 2, true>>(g, st);
        case 5: return launch_grouped<GemmCfg<32, 128, 128, 1, 4, false, 0, 2, true>>(g, st);
        case 6: return launch_grouped<GemmCfg<256, 256, 128, 2, 4, false, 0, 1, true>>(g, st);
        case 7: return launch_grouped<GemmCfg<128, 256, 128, 2, 4, false, 0, 1, true>>(g, st);
        case 8: return launch_grouped<GemmCfg<128, 128, 128, 2, 4, false, 0, 1, true>>(g, st);
        case 9: return launch_grouped<GemmCfg<192, 128, 128, 2, 4, false, 0, 1, true>>(g, st);
        case 10: return launch_grouped<GemmCfg<256, 128, 128, 4, 2, false, 0, 1, true>>(g, st);
    }
    return LLMQ_ERR_SHAPE;
}

extern "C" int llmq_gemm_w8a8_grouped_force_plan(int cfg) {
    if (cfg >= 0 && (cfg < 4 || cfg >= kNumShapes + kNumGroupedRows)) return LLMQ_ERR_SHAPE;
    forced = cfg < 0 ? -1 : cfg;
    return LLMQ_OK;
}
