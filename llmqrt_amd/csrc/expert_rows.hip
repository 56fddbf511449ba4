// Rows to their experts and back.
//
//   dispatch  place[t, j] = #{ids of a smaller expert} + #{ids of the same expert before (t, j)}        offsets[e] = #{ids of an expert below e}
//             row place[t, j] of the output is token t: as it is, in int8 with a scale per token, or in e4m3 with a scale per 128 channels
//   combine   out[t] = sum_j w[t, j] y[place[t, j]] (+ shared[t])
// Ids are counted from `first`; those outside [first, first + experts) go nowhere: they have no place (-1) and are not counted.
//
// The order is that of a stable sort, so it is the same every time.  A token is read and quantized once and written top_k times.  HBM-bound.
#include <algorithm>

#include "expert_tiles.h"
#include "llmq_common.h"
#include "quant_math.h"

namespace llmq {
namespace {

enum { OUT_SAME = LLMQ_NORM_SAME, OUT_I8 = LLMQ_NORM_I8_TOKEN, OUT_GROUP = LLMQ_NORM_FP8_GROUP };
constexpr int kMaxTop = 64, kMaxExperts = 4096;
constexpr int kMaxChunks = 2048;     // of ids
constexpr int64_t kCountAll = 2048;  // up to so many ids every token counts all of them for itself

struct DispatchArgs {
    const uint16_t* x;
    const int32_t* ids;
    const int32_t* base;  // [experts, chunks]: place of the first id of an expert in a chunk of ids; null: every token counts all ids
    void* rows;
    float* scale;
    int32_t *offsets, *places;
    int64_t ldx, K;
    int t0, ids_total;  // t0: token of block 0
    int tokens, top, first, experts, chunks, chunk_tokens;  // tokens: of this launch
};

__device__ __forceinline__ int wave_total(int v) { return __builtin_amdgcn_readlane(wave_prefix(v), kWave - 1); }

// Exclusive prefix sums of n values in LDS, in place, by NT threads; returns the total.
template <int NT>
__device__ __forceinline__ int scan_lds(int32_t* v, int n, int32_t* sums) {
    const int per = (n + NT - 1) / NT, b = threadIdx.x * per, lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
    int own = 0;
    for (int i = b; i < min(n, b + per); i++) own += v[i];
    const int upto = wave_prefix(own);
    if (lane == kWave - 1) sums[wave] = upto;
    __syncthreads();
    int before = upto - own, total = 0;
    for (int w = 0; w < NT / kWave; w++) {
        if (w < wave) before += sums[w];
        total += sums[w];
    }
    for (int i = b; i < min(n, b + per); i++) {
        const int x = v[i];
        v[i] = before, before += x;
    }
    __syncthreads();
    return total;
}

// A block per expert: how many ids go to smaller experts, and how many of its own each chunk of ids holds.
__global__ __launch_bounds__(1024) void expert_bases_kernel(const int32_t* __restrict__ ids, int n, int first, int experts, int chunk, int chunks,
                                                            int32_t* __restrict__ base, int32_t* __restrict__ offsets) {
    __shared__ int32_t same[kMaxChunks], sums[1024 / kWave], s_less[1024 / kWave];
    const int e = blockIdx.x, lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
    int less = 0;
    for (int c = wave; c < chunks; c += 1024 / kWave) {
        const int lo = c * chunk, hi = min(n - lo, chunk) + lo;
        int mine = 0;
#pragma unroll 4
        for (int i = lo + lane; i < hi; i += kWave) {
            const uint32_t v = (uint32_t)ids[i] - (uint32_t)first;
            mine += v == (uint32_t)e, less += v < (uint32_t)e;
        }
        mine = wave_total(mine);
        if (lane == 0) same[c] = mine;
    }
    less = wave_total(less);
    if (lane == 0) s_less[wave] = less;
    __syncthreads();
    const int own = scan_lds<1024>(same, chunks, sums);
    less = 0;
    for (int w = 0; w < 1024 / kWave; w++) less += s_less[w];
    for (int c = threadIdx.x; c < chunks; c += 1024) base[(int64_t)e * chunks + c] = less + same[c];
    if (threadIdx.x == 0) {
        offsets[e] = less;
        if (e == experts - 1) offsets[experts] = less + own;
    }
}

// A block per token.  ALL: every token counts all ids for itself, and one more block counts them for the offsets.  NC > 0: the row stays in NC registers per thread; 0: rows of any
// length, read again for every copy.
template <int DT, int OUT, bool ALL, int NC, int NT>
__global__ __launch_bounds__(NT) void dispatch_kernel(DispatchArgs a) {
    constexpr int NW = NT / kWave, REGS = NC > 0 ? NC : 1, JW = 4;
    __shared__ float smem[NW];
    __shared__ int32_t place[kMaxTop];
    const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(tid / kWave);
    if constexpr (ALL) if (blockIdx.x == (unsigned)a.tokens) {  // block-uniform
        __shared__ int32_t count[kMaxExperts], sums[NW];
        for (int e = tid; e < a.experts; e += NT) count[e] = 0;
        __syncthreads();
        for (int i = tid; i < a.ids_total; i += NT) {
            const uint32_t e = (uint32_t)a.ids[i] - (uint32_t)a.first;
            if (e < (uint32_t)a.experts) atomicAdd(&count[e], 1);
        }
        __syncthreads();
        const int total = scan_lds<NT>(count, a.experts, sums);
        for (int e = tid; e < a.experts; e += NT) a.offsets[e] = count[e];
        if (tid == 0) a.offsets[a.experts] = total;
        return;
    }
    const int t = a.t0 + (int)blockIdx.x;
    const int nchunk = (int)(a.K >> 3);
    const uint4* xr = reinterpret_cast<const uint4*>(a.x + (int64_t)t * a.ldx);
    uint4 v[REGS];
    if (NC > 0) {
#pragma unroll
        for (int c = 0; c < NC; c++) v[c] = tid + c * NT < nchunk ? xr[tid + c * NT] : make_uint4(0, 0, 0, 0);
    }

    // ---- places of the token's copies: JW of them per wavefront and pass over the ids
    const int mine = t * a.top, chunk = ALL ? 0 : t / a.chunk_tokens, lo = ALL ? 0 : chunk * a.chunk_tokens * a.top;
    for (int j0 = wave * JW; j0 < a.top; j0 += NW * JW) {
        uint32_t e[JW];
        int n[JW];
#pragma unroll
        for (int k = 0; k < JW; k++) {
            e[k] = j0 + k < a.top ? (uint32_t)a.ids[mine + j0 + k] - (uint32_t)a.first : ~0u;
            n[k] = 0;
        }
        if (!ALL) {
#pragma unroll 4
            for (int i = lo + lane; i < mine + a.top; i += kWave) {
                const uint32_t id = (uint32_t)a.ids[i] - (uint32_t)a.first;
#pragma unroll
                for (int k = 0; k < JW; k++) n[k] += id == e[k] && i < mine + j0 + k;
            }
        } else {
#pragma unroll 4
            for (int i = lane; i < a.ids_total; i += kWave) {
                const uint32_t id = (uint32_t)a.ids[i] - (uint32_t)a.first;
#pragma unroll
                for (int k = 0; k < JW; k++) n[k] += id < e[k] || (id == e[k] && i < mine + j0 + k);
            }
        }
#pragma unroll
        for (int k = 0; k < JW; k++) {
            if (j0 + k >= a.top) break;
            const bool goes = e[k] < (uint32_t)a.experts;
            int p = wave_total(n[k]);
            if (!ALL && goes) p += a.base[(int64_t)e[k] * a.chunks + chunk];
            if (!goes) p = -1;
            if (lane == 0) place[j0 + k] = p, a.places[mine + j0 + k] = p;
        }
    }
    __syncthreads();

    // ---- the row, in its output's form, to every place
    if (OUT == OUT_SAME) {
        for (int j = 0; j < a.top; j++) {
            const int p = place[j];
            if (p < 0) continue;
            uint4* to = reinterpret_cast<uint4*>((uint16_t*)a.rows + (int64_t)p * a.K);
            if (NC > 0) {
#pragma unroll
                for (int c = 0; c < NC; c++)
                    if (tid + c * NT < nchunk) to[tid + c * NT] = v[c];
            } else {
                for (int i = tid; i < nchunk; i += NT) to[i] = xr[i];
            }
        }
        return;
    }
    if (OUT == OUT_I8) {  // the scale and the quotients are values of x's type, as in llmq_quant_i8_per_token
        float amax = 0.f;
        if (NC > 0) {
#pragma unroll
            for (int c = 0; c < NC; c++) amax = max_nonneg(amax, absmax8(v[c], DT == LLMQ_BF16));
        } else {
            for (int i = tid; i < nchunk; i += NT) amax = max_nonneg(amax, absmax8(xr[i], DT == LLMQ_BF16));
        }
        amax = block_max<NW>(amax, smem);
        const float s = scale_from_amax<DT, MODE_I8>(amax), inv_s = 1.0f / s;
        const bool fin = amax < __builtin_inff() && s > 0.f;
        auto codes = [&](uint4 r) __attribute__((always_inline)) {
            return fin ? quant8<DT, MODE_I8, Q_DT, true>(r, s, inv_s) : quant8<DT, MODE_I8, Q_DT, false>(r, s, inv_s);
        };
        uint2 q[REGS];
        if (NC > 0) {
#pragma unroll
            for (int c = 0; c < NC; c++) q[c] = codes(v[c]);
        }
        for (int j = 0; j < a.top; j++) {
            const int p = place[j];
            if (p < 0) continue;
            uint2* to = reinterpret_cast<uint2*>((uint8_t*)a.rows + (int64_t)p * a.K);
            if (tid == 0) a.scale[p] = s;
            if (NC > 0) {
#pragma unroll
                for (int c = 0; c < NC; c++)
                    if (tid + c * NT < nchunk) to[tid + c * NT] = q[c];
            } else {
                for (int i = tid; i < nchunk; i += NT) to[i] = codes(xr[i]);
            }
        }
        return;
    }
    // a scale per 16 chunks, which 16 neighbouring lanes hold
    const int groups = (nchunk + kTeam - 1) / kTeam;
    auto group_codes = [&](uint4 r, float& s) __attribute__((always_inline)) {
        const float amax = team_max(absmax8(r, DT == LLMQ_BF16));
        s = scale32<MODE_F8>(amax);
        const float inv_s = 1.0f / s;
        float f[8];
        widen8<DT>(r, f);
        return __all(near_ok(amax, s)) ? codes8<MODE_F8, true>(f, s, inv_s) : codes8<MODE_F8, false>(f, s, inv_s);
    };
    uint2 q[REGS];
    float s[REGS];
    if (NC > 0) {
#pragma unroll
        for (int c = 0; c < NC; c++) q[c] = group_codes(v[c], s[c]);
    }
    for (int j = 0; j < a.top; j++) {
        const int p = place[j];
        if (p < 0) continue;  // block-uniform
        uint2* to = reinterpret_cast<uint2*>((uint8_t*)a.rows + (int64_t)p * a.K);
        float* ts = a.scale + (int64_t)p * groups;
        if (NC > 0) {
#pragma unroll
            for (int c = 0; c < NC; c++) {
                const int i = tid + c * NT;
                if (i < nchunk) to[i] = q[c];
                if (i < nchunk && i % kTeam == 0) ts[i / kTeam] = s[c];
            }
        } else {
            for (int b = 0; b < nchunk; b += NT) {
                const int i = b + tid;
                const uint2 c = group_codes(i < nchunk ? xr[i] : make_uint4(0, 0, 0, 0), s[0]);
                if (i < nchunk) to[i] = c;
                if (i < nchunk && i % kTeam == 0) ts[i / kTeam] = s[0];
            }
        }
    }
}

// ids per chunk, a whole number of tokens' (0: every token counts all ids)
int64_t chunk_tokens(int64_t tokens, int64_t top) {
    if (tokens * top <= kCountAll) return 0;
    const int64_t least = (tokens + kMaxChunks - 1) / kMaxChunks;
    return std::max(least, std::max<int64_t>(1, 512 / top));
}

template <int DT, int OUT, bool ALL>
int launch_dispatch(const DispatchArgs& a, unsigned grid, hipStream_t st) {
    const int64_t chunks = a.K >> 3;
#define LLMQ_DISPATCH(NC, NT) hipLaunchKernelGGL((dispatch_kernel<DT, OUT, ALL, NC, NT>), dim3(grid), dim3(NT), 0, st, a)
    if (chunks <= 128) LLMQ_DISPATCH(1, 128);
    else if (chunks <= 256) LLMQ_DISPATCH(1, 256);
    else if (chunks <= 512) LLMQ_DISPATCH(2, 256);
    else if (chunks <= 1024) LLMQ_DISPATCH(4, 256);
    else if (chunks <= 2560) LLMQ_DISPATCH(5, 512);
    else LLMQ_DISPATCH(0, 512);
#undef LLMQ_DISPATCH
    return launch_status();
}
template <int DT>
int launch_dispatch_out(int out, const DispatchArgs& a, unsigned grid, hipStream_t st) {
    switch (out) {
        case OUT_SAME: return a.base ? launch_dispatch<DT, OUT_SAME, false>(a, grid, st) : launch_dispatch<DT, OUT_SAME, true>(a, grid, st);
        case OUT_I8: return a.base ? launch_dispatch<DT, OUT_I8, false>(a, grid, st) : launch_dispatch<DT, OUT_I8, true>(a, grid, st);
        default: return a.base ? launch_dispatch<DT, OUT_GROUP, false>(a, grid, st) : launch_dispatch<DT, OUT_GROUP, true>(a, grid, st);
    }
}

// ---- combine
struct CombineArgs {
    const uint16_t* y;
    const int32_t* places;
    const float* weights;
    const uint16_t* shared;
    uint16_t* out;
    int64_t ldy, lds, rows, total;  // total: chunks of 8 channels of the output
    uint32_t chunks;                // of a row
    int top;
};

// A thread per chunk, four rows requested before the first is used.
template <int DT>
__global__ __launch_bounds__(256) void combine_kernel(CombineArgs a) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= a.total) return;
    const int64_t t = i <= 0xffffffffLL ? (uint32_t)i / a.chunks : i / a.chunks;
    const int64_t c = (i - t * a.chunks) * 8;
    float acc[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    for (int j0 = 0; j0 < a.top; j0 += 4) {
        uint4 v[4];
        float w[4];
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const int j = j0 + k;
            const int64_t p = j < a.top ? a.places[t * a.top + j] : -1;
            const bool has = p >= 0 && p < a.rows;
            w[k] = has ? a.weights[t * a.top + j] : 0.f;
            v[k] = has ? *reinterpret_cast<const uint4*>(a.y + p * a.ldy + c) : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int k = 0; k < 4; k++) {
            float f[8];
            widen8<DT>(v[k], f);
#pragma unroll
            for (int e = 0; e < 8; e++) acc[e] = fmaf(w[k], f[e], acc[e]);
        }
    }
    if (a.shared) {
        float f[8];
        widen8<DT>(*reinterpret_cast<const uint4*>(a.shared + t * a.lds + c), f);
#pragma unroll
        for (int e = 0; e < 8; e++) acc[e] += f[e];
    }
    *reinterpret_cast<uint4*>(a.out + t * (int64_t)a.chunks * 8 + c) = narrow8<DT>(acc);
}

bool aligned8(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 7u) == 0; }

}  // namespace
}  // namespace llmq

using namespace llmq;

extern "C" size_t llmq_dispatch_workspace_bytes(int64_t tokens, int64_t top_k, int64_t experts) {
    if (tokens <= 0 || top_k <= 0 || top_k > kMaxTop || experts <= 0 || experts > kMaxExperts || tokens > 0x7fffff00LL / top_k) return 0;
    const int64_t per = chunk_tokens(tokens, top_k);
    return per ? (size_t)(experts * ((tokens + per - 1) / per) * 4) : 0;
}

extern "C" int llmq_dispatch_experts(int out, const void* x, int x_dtype, int64_t tokens, int64_t K, int64_t ldx, const int32_t* ids, int64_t top_k,
                                     int64_t first_expert, int64_t experts, void* rows, float* scale, int32_t* offsets, int32_t* places,
                                     void* workspace, size_t workspace_bytes, llmq_stream_t stream) {
    if ((out != OUT_SAME && out != OUT_I8 && out != OUT_GROUP) || (x_dtype != LLMQ_BF16 && x_dtype != LLMQ_F16)) return LLMQ_ERR_DTYPE;
    if (tokens < 0 || K < 0 || K > 0x7fffffffLL || ldx < K || (K & 7) || (ldx & 7) || top_k < 1 || top_k > kMaxTop || experts < 1 ||
        experts > kMaxExperts || first_expert < 0 || first_expert > 0x7fff0000LL || tokens > 0x7fffff00LL / top_k)
        return LLMQ_ERR_SHAPE;
    if (!offsets || (tokens > 0 && (!ids || !places || (K > 0 && (!x || !rows || (out != OUT_SAME && !scale)))))) return LLMQ_ERR_NULL;
    if (tokens > 0 && K == 0) return LLMQ_ERR_SHAPE;
    if (tokens > 0 && (!aligned16(x) || (out == OUT_SAME ? !aligned16(rows) : !aligned8(rows)))) return LLMQ_ERR_ALIGN;
    const size_t need = llmq_dispatch_workspace_bytes(tokens, top_k, experts);
    if (need && (!workspace || workspace_bytes < need)) return LLMQ_ERR_WORKSPACE;
    if (need && (reinterpret_cast<uintptr_t>(workspace) & 3u)) return LLMQ_ERR_ALIGN;
    DispatchArgs a = {};
    a.x = (const uint16_t*)x, a.ids = ids, a.rows = rows, a.scale = scale, a.offsets = offsets, a.places = places;
    a.ldx = ldx, a.K = K, a.ids_total = (int)(tokens * top_k), a.top = (int)top_k, a.first = (int)first_expert, a.experts = (int)experts;
    const hipStream_t st = (hipStream_t)stream;
    const int64_t per = chunk_tokens(tokens, top_k);
    if (per) {
        a.chunk_tokens = (int)per, a.chunks = (int)((tokens + per - 1) / per), a.base = (const int32_t*)workspace;
        hipLaunchKernelGGL(expert_bases_kernel, dim3((unsigned)experts), dim3(1024), 0, st, ids, a.ids_total, a.first, a.experts, (int)(per * top_k), a.chunks,
                           (int32_t*)workspace, offsets);
        if (launch_status() != LLMQ_OK) return LLMQ_ERR_LAUNCH;
    }
    const int64_t step = (int64_t)1 << 21;  // tokens of a grid: 2^32 threads are too many
    int rc = LLMQ_OK;
    for (int64_t t = 0; rc == LLMQ_OK && (t < tokens || (t == 0 && !per)); t += step) {
        a.t0 = (int)t, a.tokens = (int)std::min(step, tokens - t);
        const unsigned grid = (unsigned)a.tokens + (per ? 0 : 1);  // (every token counts all ids: one launch, with the block for the offsets)
        rc = x_dtype == LLMQ_BF16 ? launch_dispatch_out<LLMQ_BF16>(out, a, grid, st) : launch_dispatch_out<LLMQ_F16>(out, a, grid, st);
    }
    return rc;
}

extern "C" int llmq_combine_experts(const void* y, int dtype, int64_t rows, int64_t N, int64_t ldy, const int32_t* places, const float* weights,
                                    int64_t tokens, int64_t top_k, const void* shared, int64_t ld_shared, void* out, llmq_stream_t stream) {
    if (dtype != LLMQ_BF16 && dtype != LLMQ_F16) return LLMQ_ERR_DTYPE;
    if (rows < 0 || tokens < 0 || N < 0 || N > 0x7fffffffLL || (N & 7) || ldy < N || (ldy & 7) || top_k < 1 || top_k > kMaxTop ||
        tokens > 0x7fffff00LL / top_k || (shared && (ld_shared < N || (ld_shared & 7))))
        return LLMQ_ERR_SHAPE;
    if (tokens == 0 || N == 0) return LLMQ_OK;
    if ((rows > 0 && !y) || !places || !weights || !out) return LLMQ_ERR_NULL;
    if (!aligned16(y) || !aligned16(out) || (shared && !aligned16(shared))) return LLMQ_ERR_ALIGN;
    const int64_t step = std::max<int64_t>(1, ((int64_t)1 << 31) / (N / 8));  // tokens of a grid of fewer than 2^32 threads
    int rc = LLMQ_OK;
    for (int64_t t = 0; t < tokens && rc == LLMQ_OK; t += step) {
        CombineArgs a = {};
        a.y = (const uint16_t*)y, a.places = places + t * top_k, a.weights = weights + t * top_k, a.out = (uint16_t*)out + t * N;
        if (shared) a.shared = (const uint16_t*)shared + t * ld_shared;
        a.ldy = ldy, a.lds = ld_shared, a.rows = rows, a.chunks = (uint32_t)(N / 8), a.total = std::min(step, tokens - t) * a.chunks, a.top = (int)top_k;
        const dim3 grid((unsigned)((a.total + 255) / 256));
        if (dtype == LLMQ_BF16) hipLaunchKernelGGL((combine_kernel<LLMQ_BF16>), grid, dim3(256), 0, (hipStream_t)stream, a);
        else hipLaunchKernelGGL((combine_kernel<LLMQ_F16>), grid, dim3(256), 0, (hipStream_t)stream, a);
        rc = launch_status();
    }
    return rc;
}
