// W8A8 product by experts: the int8 tile kernel of gemm_tile_impl.h over rows that are sorted by expert.
//
//   out[m, n] = dtype( (acc[m, n] a_scale[m]) w_scale[e, n] + bias[e, n] ),  acc[m, n] = sum_k A[m, k] B[e, n, k],  m of expert e
//
// The host does not know the experts' rows, so the grid is what any distribution can need (each expert may end with a tile that is not full) and a block
// finds its tile from the offsets.
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

thread_local int forced = -1;

// Tiles of 256 rows where the experts have them on average, of 32 where they have a few.
int plan(int64_t M, int64_t experts) {
    const int64_t rows = M / std::max<int64_t>(1, std::min(M, experts));
    return rows > 192 ? 6 : rows > 48 ? 7 : rows > 24 ? 4 : 5;
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
    const int cfg = forced >= 0 && (forced < kNumShapes || experts <= kGroupedRowsExperts) ? forced : plan(M, experts);
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
