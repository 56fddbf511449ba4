// Gated activation between two products, with an output in 16 or 8 bits.
//
//   y[m, k] = g / (1 + exp(-g)) * u,   g = x[m, k], u = x[m, N + k]
//   and y rounded once to x_dtype, or quantized:  int8 s = max(max_k |y|, 1e-5) / 127,  q = rint(y / s)
//                                                 e4m3 s = max(max |y|, 1e-12) / 448, per token or per token and group of 128 channels
// Everything between x and the codes is fp32.  HBM-bound: 4 bytes read and 1 or 2 written per output; a few rows are a launch and a chain of latencies (37 x 18944
// int8 4.9 us: two loads, the formula, a maximum over 16 wavefronts, the codes).
#include <algorithm>

#include "llmq_common.h"
#include "quant_math.h"

namespace llmq {
namespace {

enum { OUT_SAME = LLMQ_NORM_SAME, OUT_I8 = LLMQ_NORM_I8_TOKEN, OUT_F8 = LLMQ_NORM_FP8_TOKEN, OUT_GROUP = LLMQ_NORM_FP8_GROUP };
constexpr int kSiluThreads = 256;

struct SiluArgs {
    const uint16_t* x;
    uint16_t* y;  // OUT_SAME
    uint8_t* q;   // otherwise
    float* scale;
    int64_t ldx, M, N;
};

// exp by the base-2 instruction: y is off by (2 |g| + 8) 2^-24 of itself.  g of -inf gives -inf * 0 = NaN, as the formula does.
__device__ __forceinline__ float silu(float g) {
    return g * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-1.44269504088896f * g));
}
// Below -87 the reciprocal, below -88 exp(-g) itself leaves the range of fp32, while y still has bits where u is large.  From kFarGate on 1 is nothing beside exp(-g),
// which is taken 2^-126 of, and u as well: y is then 0 only where it is less than 3e-74 |u| (g below -174).
constexpr float kFarGate = -80.0f;
__device__ __forceinline__ float far_silu_mul(float g, float u) {
    return g * __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(-1.44269504088896f * g - 126.0f)) * (u * 0x1p-126f);
}
template <int DT>
__device__ __forceinline__ void gated8(uint4 gv, uint4 uv, float* y) {
    float g[8], u[8];
    widen8<DT>(gv, g), widen8<DT>(uv, u);
    uint32_t most = 0;  // of negative numbers, the bits of the lowest
#pragma unroll
    for (int i = 0; i < 8; i++) y[i] = silu(g[i]) * u[i], most = max(most, __float_as_uint(g[i]));
    if (__any(most > __float_as_uint(kFarGate)))  // uniform, and rare
#pragma unroll
        for (int i = 0; i < 8; i++) y[i] = g[i] < kFarGate ? far_silu_mul(g[i], u[i]) : y[i];
}

// No reduction over the whole row: 16 lanes take 128 channels of a row, 8 of each half a lane.  One such piece per lane, and many blocks: with two or four
// in flight per lane, 8192 x 18944 takes 144 and 154 us by groups where one takes 134 (5.8 TB/s), 37 x 18944 3.1 and 4.4 where 2.7.
template <int DT, bool GROUP>
__global__ __launch_bounds__(kSiluThreads) void silu_groups_kernel(SiluArgs a, uint32_t groups, uint32_t total) {
    const int l = threadIdx.x % kTeam;
    const uint32_t g = blockIdx.x * (kSiluThreads / kTeam) + threadIdx.x / kTeam, row = g / groups;
    const int64_t k = (int64_t)(g - row * groups) * 128 + l * 8;
    const bool in = g < total && k < a.N;
    const uint16_t* xr = a.x + (int64_t)row * a.ldx + k;
    const uint4 gv = in ? *reinterpret_cast<const uint4*>(xr) : make_uint4(0, 0, 0, 0);
    const uint4 uv = in ? *reinterpret_cast<const uint4*>(xr + a.N) : make_uint4(0, 0, 0, 0);
    const int64_t to = (int64_t)row * a.N + k;
    float y[8];
    gated8<DT>(gv, uv, y);
    if (!GROUP) {
        if (in) *reinterpret_cast<uint4*>(a.y + to) = narrow8<DT>(y);
        return;
    }
    const float amax = team_max(absmax8f(y)), s = scale32<MODE_F8>(amax), inv_s = 1.0f / s;
    uint2 c;
    if (__all(near_ok(amax, s))) c = codes8<MODE_F8, true>(y, s, inv_s);
    else c = codes8<MODE_F8, false>(y, s, inv_s);
    if (in) *reinterpret_cast<uint2*>(a.q + to) = c;
    if (l == 0 && g < total) a.scale[g] = s;
}

// A scale per row.  NT threads per row, RPB rows per block (more than one: within a wavefront each, and no barrier).  NC > 0: a row's outputs stay in 8 NC
// registers per thread between the maximum and the codes; 0: rows of any length, computed twice.
template <int DT, int MODE, int NC, int NT, int RPB>
__global__ __launch_bounds__(NT * RPB) void silu_rows_kernel(SiluArgs a) {
    static_assert(RPB == 1 ? NT >= kWave : NT == 16 || NT == 32 || NT == kWave, "several rows per block are within a wavefront each");
    __shared__ float smem[RPB > 1 ? 1 : NT / kWave];
    const int tid = threadIdx.x % NT;
    const int64_t own = (int64_t)blockIdx.x * RPB + threadIdx.x / NT, row = RPB > 1 ? min(own, a.M - 1) : own;
    const int nchunk = RPB > 1 && own >= a.M ? 0 : (int)(a.N >> 3);  // (lanes without a row have no chunks)
    const uint4* gr = reinterpret_cast<const uint4*>(a.x + row * a.ldx);
    const uint4* ur = reinterpret_cast<const uint4*>(a.x + row * a.ldx + a.N);
    uint2* qr = reinterpret_cast<uint2*>(a.q + row * a.N);
    float y[NC > 0 ? NC : 1][8], amax = 0.f;
    if (NC > 0) {
        uint4 gv[NC > 0 ? NC : 1], uv[NC > 0 ? NC : 1];
#pragma unroll
        for (int c = 0; c < NC; c++) {
            const int i = tid + c * NT;
            gv[c] = i < nchunk ? gr[i] : make_uint4(0, 0, 0, 0);
            uv[c] = i < nchunk ? ur[i] : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int c = 0; c < NC; c++) {
            gated8<DT>(gv[c], uv[c], y[c]);
            amax = max_nonneg(amax, absmax8f(y[c]));
        }
    } else {
        for (int i = tid; i < nchunk; i += NT) {
            gated8<DT>(gr[i], ur[i], y[0]);
            amax = max_nonneg(amax, absmax8f(y[0]));
        }
    }
    if constexpr (RPB == 1) {
        amax = block_max<NT / kWave>(amax, smem);
    } else {
        amax = NT == kWave ? wave_max(amax) : team_max(amax);
        if constexpr (NT == 32) amax = max_nonneg(amax, lane_xor<16>(amax));
    }
    const float s = scale32<MODE>(amax), inv_s = 1.0f / s;
    if (tid == 0 && (RPB == 1 || own < a.M)) a.scale[row] = s;
    const bool fast = near_ok(amax, s);  // of the row
    if (NC > 0) {
#pragma unroll
        for (int c = 0; c < NC; c++) {
            const int i = tid + c * NT;
            if (i < nchunk) qr[i] = fast ? codes8<MODE, true>(y[c], s, inv_s) : codes8<MODE, false>(y[c], s, inv_s);
        }
    } else {
        for (int i = tid; i < nchunk; i += NT) {
            gated8<DT>(gr[i], ur[i], y[0]);
            qr[i] = fast ? codes8<MODE, true>(y[0], s, inv_s) : codes8<MODE, false>(y[0], s, inv_s);
        }
    }
}

template <int DT, bool GROUP>
int launch_groups(const SiluArgs& a, hipStream_t st) {
    constexpr int TEAMS = kSiluThreads / kTeam;
    const uint32_t groups = (uint32_t)((a.N + 127) / 128), total = (uint32_t)(a.M * groups);
    hipLaunchKernelGGL((silu_groups_kernel<DT, GROUP>), dim3((total + TEAMS - 1) / TEAMS), dim3(kSiluThreads), 0, st, a, groups, total);
    return launch_status();
}

// Two chunks per thread until a row takes 1024 of them: fewer threads per row mean less to wait for between the maximum and the codes, fewer chunks more
// wavefronts that hide it.  Up to 64 threads, rows share a wavefront and a block of 256 threads.  32768 rows in int8, us, threads x chunks: 256 channels 16 x 2
// 8.8, 32 x 2 10.4, 64 x 1 18.8; 512 32 x 2 16.7, 64 x 2 18.5; 552 64 x 2 21.8, 32 x 3 19.0, 768 23.6 and 24.3.  8192 rows: 1024 channels 64 x 2 9.2, 128 x 1
// 11.9, 256 x 1 14.4; 2048 128 x 2 17.0, 64 x 4 17.8, 256 x 1 20.7; 3584 256 x 2 28.0, 512 x 1 34.1; 8192 512 x 2 62.9, 1024 x 1 73.7, 256 x 4 64.1; 13696 1024
// x 2 96, 512 x 4 105; 18944 1024 x 3 136, 512 x 5 145; 28672 1024 x 4 221, rows computed twice 294.  A few rows of 8192: 512 x 2 2.9, 1024 x 1 3.5.
template <int DT, int MODE>
int launch_rows(const SiluArgs& a, hipStream_t st) {
    const int64_t chunks = a.N >> 3;
#define LLMQ_SILU(NC, NT, RPB) \
    hipLaunchKernelGGL((silu_rows_kernel<DT, MODE, NC, NT, RPB>), dim3((unsigned)((a.M + RPB - 1) / RPB)), dim3(NT * RPB), 0, st, a)
    if (chunks <= 32) LLMQ_SILU(2, 16, 16);
    else if (chunks <= 64) LLMQ_SILU(2, 32, 8);
    else if (chunks <= 128) LLMQ_SILU(2, 64, 4);
    else if (chunks <= 256) LLMQ_SILU(2, 128, 1);
    else if (chunks <= 512) LLMQ_SILU(2, 256, 1);
    else if (chunks <= 1024) LLMQ_SILU(2, 512, 1);
    else if (chunks <= 2048) LLMQ_SILU(2, 1024, 1);
    else if (chunks <= 3 * 1024) LLMQ_SILU(3, 1024, 1);
    else if (chunks <= 4096) LLMQ_SILU(4, 1024, 1);
    else LLMQ_SILU(0, 1024, 1);
#undef LLMQ_SILU
    return launch_status();
}

template <int DT>
int launch_silu(int out, const SiluArgs& a, hipStream_t st) {
    switch (out) {
        case OUT_SAME: return launch_groups<DT, false>(a, st);
        case OUT_GROUP: return launch_groups<DT, true>(a, st);
        case OUT_I8: return launch_rows<DT, MODE_I8>(a, st);
        default: return launch_rows<DT, MODE_F8>(a, st);
    }
}

}  // namespace
}  // namespace llmq

using namespace llmq;

extern "C" int llmq_silu_mul(int out, const void* x, int x_dtype, int64_t M, int64_t N, int64_t ldx, void* y, float* scale, llmq_stream_t stream) {
    if (out < OUT_SAME || out > OUT_GROUP || (x_dtype != LLMQ_BF16 && x_dtype != LLMQ_F16)) return LLMQ_ERR_DTYPE;
    if (M < 0 || N < 0 || M > 0x7fffffffLL || N > 0x3fffffffLL || ldx < 2 * N || (N & 7) || (ldx & 7)) return LLMQ_ERR_SHAPE;
    if (M == 0 || N == 0) return LLMQ_OK;
    if (!x || !y || (out != OUT_SAME && !scale)) return LLMQ_ERR_NULL;
    if (!aligned16(x) || (out == OUT_SAME ? !aligned16(y) : (reinterpret_cast<uintptr_t>(y) & 7u) != 0)) return LLMQ_ERR_ALIGN;
    // a grid holds fewer than 2^32 threads: rows beyond that many go to further launches
    const int64_t groups = (N + 127) / 128, per_row = out == OUT_GROUP ? groups : 1;
    const int64_t step = out == OUT_SAME || out == OUT_GROUP ? std::max<int64_t>(1, ((int64_t)1 << 27) / groups) : (int64_t)1 << 21;
    int rc = LLMQ_OK;
    for (int64_t m = 0; m < M && rc == LLMQ_OK; m += step) {
        SiluArgs a = {};
        a.x = (const uint16_t*)x + m * ldx, a.ldx = ldx, a.M = std::min(step, M - m), a.N = N;
        if (out == OUT_SAME) a.y = (uint16_t*)y + m * N;
        else a.q = (uint8_t*)y + m * N, a.scale = scale + m * per_row;
        rc = x_dtype == LLMQ_BF16 ? launch_silu<LLMQ_BF16>(out, a, (hipStream_t)stream) : launch_silu<LLMQ_F16>(out, a, (hipStream_t)stream);
    }
    return rc;
}
