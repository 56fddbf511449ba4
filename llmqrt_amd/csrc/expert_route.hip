// Routing: a token's experts and their weights from its scores.
//
//   s = softmax(l) or 1 / (1 + exp(-l));  c = s + bias;  experts = the top_k largest c, ties to the lowest expert;  weights = s of those, divided by their
//   sum if asked for, times a factor
// Groups: of neighbouring experts; only the top_groups groups with the largest score (max c, or the sum of the two largest c) take part.
// l or bias of -inf: the expert is masked, never chosen.  A place that is left over has expert -1 and weight 0.
//
// Which experts are chosen has to follow from the scores, not from how they were rounded: without a bias the order of c is that of the logits, which are
// compared as they are; with one, and where two scores of a group are added, scores are formed and compared in 64 bits.
//
// LPT lanes share a token, V neighbouring experts each, in registers.  A choice is the maximum of the lanes' best ones by lane selects; the lane that had it
// notes it in LDS and looks for its next one.
#include <algorithm>
#include <type_traits>

#include "llmq_common.h"

namespace llmq {
namespace {

constexpr int kThreads = 256, kMaxTop = 64, kMaxExperts = 1024, kMaxGroups = 64;

struct RouteArgs {
    const void* logits;
    const float* bias;
    float* weights;
    int32_t* ids;
    int64_t ld, tokens;
    int experts, top, groups, top_groups, group_size;
    int sigmoid, top2, renormalize;
    float scale;
};

// the value of lane (lane ^ O) of a wavefront
template <int O>
__device__ __forceinline__ uint32_t from_lane(uint32_t v) {
    if constexpr (O == 32) {
        float a, b;
        lane_xor32_pair(__uint_as_float(v), a, b);
        return (threadIdx.x & 32) ? __float_as_uint(a) : __float_as_uint(b);
    } else {
        return __float_as_uint(lane_xor<O>(__uint_as_float(v)));
    }
}
template <int LPT, class T, class F>
__device__ __forceinline__ T team_reduce(T v, F&& f) {
    auto step = [&](auto o_c) __attribute__((always_inline)) {
        constexpr int O = decltype(o_c)::value;
        if constexpr (O < LPT) {
            if constexpr (sizeof(T) == 4) {
                v = f(v, __builtin_bit_cast(T, from_lane<O>(__builtin_bit_cast(uint32_t, v))));
            } else {
                const uint64_t u = __builtin_bit_cast(uint64_t, v);
                v = f(v, __builtin_bit_cast(T, (uint64_t)from_lane<O>((uint32_t)u) | (uint64_t)from_lane<O>((uint32_t)(u >> 32)) << 32));
            }
        }
    };
    step(std::integral_constant<int, 1>{}), step(std::integral_constant<int, 2>{}), step(std::integral_constant<int, 4>{});
    step(std::integral_constant<int, 8>{}), step(std::integral_constant<int, 16>{}), step(std::integral_constant<int, 32>{});
    return v;
}

// Unsigned keys in the order of the values; a NaN is above all, 0 below all (masked)
__device__ __forceinline__ uint64_t key_of(double c) {
    const uint64_t u = __builtin_bit_cast(uint64_t, c + 0.0);  // (-0 is 0)
    return c != c ? ~0ull : u >> 63 ? ~u : u | 1ull << 63;
}
__device__ __forceinline__ double value_of(uint64_t k) { return __builtin_bit_cast(double, k >> 63 ? k & ~(1ull << 63) : ~k); }
__device__ __forceinline__ uint64_t key_of(float c) {
    const uint32_t u = __float_as_uint(c + 0.0f);
    return (uint64_t)(c != c ? ~0u : u >> 31 ? ~u : u | 1u << 31) << 32;
}

__device__ __forceinline__ void wave_fence() {  // LDS written by other lanes of the wavefront
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront", "local");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront", "local");
}

template <int DT, bool EXACT, int LPT, int V>
__global__ __launch_bounds__(kThreads) void route_kernel(RouteArgs a) {
    constexpr int TPB = kThreads / LPT;
    extern __shared__ uint64_t dyn[];  // with groups: keys of the block's experts, then of its groups
    __shared__ int32_t s_id[TPB][kMaxTop];
    __shared__ float s_x[TPB][kMaxTop];
    const int tid = threadIdx.x, lane = tid & (kWave - 1), team = tid / LPT, l = tid % LPT;
    const int64_t token = (int64_t)blockIdx.x * TPB + team, t = min(token, a.tokens - 1);  // (a team without a token repeats the last one's)
    const int e0 = l * V;

    float x[V];
#pragma unroll
    for (int v = 0; v < V; v++) {
        const int64_t at = t * a.ld + e0 + v;
        x[v] = e0 + v < a.experts ? load_as_f32(a.logits, DT, at) : -__builtin_inff();
    }
    float m = x[0];
#pragma unroll
    for (int v = 1; v < V; v++) m = fmaxf(m, x[v]);
    m = team_reduce<LPT>(m, [](float p, float q) { return fmaxf(p, q); });

    uint64_t key[V];
    float sum = 1.f;  // of exp(x - m)
    if constexpr (EXACT) {
        double s[V], total = 0.0;
#pragma unroll
        for (int v = 0; v < V; v++) {
            s[v] = x[v] == -__builtin_inff() ? 0.0 : a.sigmoid ? 1.0 / (1.0 + exp(-(double)x[v])) : exp((double)x[v] - (double)m);
            total += s[v];
        }
        if (!a.sigmoid) {
            total = team_reduce<LPT>(total, [](double p, double q) { return p + q; });
            sum = (float)total;
        }
#pragma unroll
        for (int v = 0; v < V; v++) {
            const float b = a.bias && e0 + v < a.experts ? a.bias[e0 + v] : 0.f;
            const bool masked = x[v] == -__builtin_inff() || b == -__builtin_inff();
            key[v] = masked ? 0 : key_of((a.sigmoid ? s[v] : s[v] / total) + (double)b);
        }
    } else {
        if (!a.sigmoid && !a.renormalize) {
            sum = 0.f;
#pragma unroll
            for (int v = 0; v < V; v++) sum += x[v] == -__builtin_inff() ? 0.f : expf(x[v] - m);
            sum = team_reduce<LPT>(sum, [](float p, float q) { return p + q; });
        }
#pragma unroll
        for (int v = 0; v < V; v++) key[v] = x[v] == -__builtin_inff() ? 0 : key_of(x[v]);
    }

    if (a.groups > 1) {
        uint64_t* mine = dyn + team * a.experts;
        uint64_t* group = dyn + TPB * a.experts + team * a.groups;
#pragma unroll
        for (int v = 0; v < V; v++)
            if (e0 + v < a.experts) mine[e0 + v] = key[v];
        wave_fence();
        for (int g = l; g < a.groups; g += LPT) {
            uint64_t best = 0, second = 0;
            for (int i = 0; i < a.group_size; i++) {
                const uint64_t k = mine[g * a.group_size + i];
                second = k > best ? best : k > second ? k : second;
                best = k > best ? k : best;
            }
            if (EXACT && a.top2 && second != 0) best = key_of(value_of(best) + value_of(second));
            group[g] = best;
        }
        wave_fence();
#pragma unroll
        for (int v = 0; v < V; v++) {
            if (e0 + v >= a.experts) continue;
            const int g = (e0 + v) / a.group_size;
            const uint64_t k = group[g];
            int ahead = 0;
            for (int i = 0; i < a.groups; i++) ahead += group[i] > k || (group[i] == k && i < g);
            if (ahead >= a.top_groups) key[v] = 0;
        }
    }

    const uint64_t team_lanes = (LPT == 64 ? ~0ull : (1ull << LPT) - 1) << (lane / LPT * LPT);
    for (int j = 0; j < a.top; j++) {
        uint64_t best = key[0];
        int bv = 0;
#pragma unroll
        for (int v = 1; v < V; v++)
            if (key[v] > best) best = key[v], bv = v;
        const uint64_t most = team_reduce<LPT>(best, [](uint64_t p, uint64_t q) { return p > q ? p : q; });
        const uint64_t have = __ballot(best == most) & team_lanes;  // the lowest of them has the lowest expert
        if (lane == __ffsll((unsigned long long)have) - 1) {
            float bx = x[0];
#pragma unroll
            for (int v = 0; v < V; v++) {
                if (v == bv) bx = x[v], key[v] = 0;
            }
            s_id[team][j] = most ? e0 + bv : -1;
            s_x[team][j] = bx;
        }
    }
    wave_fence();

    // Weights.  Renormalised ones are ratios of the chosen scores, formed relative to the largest so that none of them underflows.
    float top_x = -__builtin_inff();
    for (int j = 0; j < a.top; j++)
        if (s_id[team][j] >= 0) top_x = fmaxf(top_x, s_x[team][j]);
    auto part = [&](float v) __attribute__((always_inline)) {
        if (!a.sigmoid) return expf(v - (a.renormalize ? top_x : m));
        if (!a.renormalize || v > 0.f || top_x > 0.f) return 1.f / (1.f + expf(-v));
        return expf(v - top_x) / (1.f + expf(v));
    };
    if (a.renormalize) {
        sum = 0.f;
        for (int j = 0; j < a.top; j++)
            if (s_id[team][j] >= 0) sum += part(s_x[team][j]);
    } else if (a.sigmoid) {
        sum = 1.f;
    }
    for (int j = l; j < a.top; j += LPT) {
        if (token >= a.tokens) break;
        const int id = s_id[team][j];
        a.ids[token * a.top + j] = id;
        a.weights[token * a.top + j] = id < 0 ? 0.f : part(s_x[team][j]) / sum * a.scale;
    }
}

template <int DT, bool EXACT>
int launch_route(const RouteArgs& a, hipStream_t st) {
    const int64_t per_team = a.groups > 1 ? (int64_t)(a.experts + a.groups) * 8 : 0;
#define LLMQ_ROUTE(LPT, V)                                                                                                          \
    hipLaunchKernelGGL((route_kernel<DT, EXACT, LPT, V>), dim3((unsigned)((a.tokens + kThreads / LPT - 1) / (kThreads / LPT))), dim3(kThreads), \
                       (unsigned)(per_team * (kThreads / LPT)), st, a)
    if (a.experts <= 64) LLMQ_ROUTE(16, 4);
    else if (a.experts <= 128) LLMQ_ROUTE(16, 8);
    else if (a.experts <= 256) LLMQ_ROUTE(32, 8);
    else LLMQ_ROUTE(64, 16);
#undef LLMQ_ROUTE
    return launch_status();
}

}  // namespace
}  // namespace llmq

using namespace llmq;

extern "C" int llmq_route_experts(int scoring, const void* logits, int logits_dtype, int64_t tokens, int64_t experts, int64_t ld, const float* bias,
                                  int64_t groups, int64_t top_groups, int group_score, int64_t top_k, int renormalize, float scale, float* weights,
                                  int32_t* ids, llmq_stream_t stream) {
    if ((scoring != LLMQ_ROUTE_SOFTMAX && scoring != LLMQ_ROUTE_SIGMOID) || (group_score != LLMQ_ROUTE_GROUP_MAX && group_score != LLMQ_ROUTE_GROUP_TOP2) ||
        (logits_dtype != LLMQ_BF16 && logits_dtype != LLMQ_F16 && logits_dtype != LLMQ_F32))
        return LLMQ_ERR_DTYPE;
    if (tokens < 0 || experts < 1 || experts > kMaxExperts || ld < experts || groups < 1 || groups > kMaxGroups || experts % groups || top_groups < 1 ||
        top_groups > groups || top_k < 1 || top_k > kMaxTop || top_k > experts / groups * top_groups || tokens > 0x7fffff00LL / top_k)
        return LLMQ_ERR_SHAPE;
    if (tokens == 0) return LLMQ_OK;
    if (!logits || !weights || !ids) return LLMQ_ERR_NULL;
    RouteArgs a = {};
    a.bias = bias, a.ld = ld, a.experts = (int)experts, a.top = (int)top_k, a.groups = (int)groups, a.top_groups = (int)top_groups;
    a.group_size = (int)(experts / groups), a.sigmoid = scoring == LLMQ_ROUTE_SIGMOID, a.top2 = group_score == LLMQ_ROUTE_GROUP_TOP2;
    a.renormalize = renormalize != 0, a.scale = scale;
    const bool exact = bias || (groups > 1 && a.top2);
    const int64_t step = (int64_t)1 << 24, size = logits_dtype == LLMQ_F32 ? 4 : 2;  // tokens of a grid: 2^32 threads are too many
    int rc = LLMQ_OK;
    for (int64_t t = 0; t < tokens && rc == LLMQ_OK; t += step) {
        a.logits = (const uint8_t*)logits + t * ld * size, a.weights = weights + t * top_k, a.ids = ids + t * top_k, a.tokens = std::min(step, tokens - t);
        const hipStream_t st = (hipStream_t)stream;
        if (logits_dtype == LLMQ_F32) rc = exact ? launch_route<LLMQ_F32, true>(a, st) : launch_route<LLMQ_F32, false>(a, st);
        else if (logits_dtype == LLMQ_BF16) rc = exact ? launch_route<LLMQ_BF16, true>(a, st) : launch_route<LLMQ_BF16, false>(a, st);
        else rc = exact ? launch_route<LLMQ_F16, true>(a, st) : launch_route<LLMQ_F16, false>(a, st);
    }
    return rc;
}
