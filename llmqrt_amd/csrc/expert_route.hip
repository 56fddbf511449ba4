// Routing: a token's experts and their weights from its scores.
//
//   s = softmax(l) or 1 / (1 + exp(-l));  c = s + bias;  experts = the top_k largest c, ties to the lowest expert;  weights = s of those, divided by their
//   sum if asked for, times a factor
// Groups: of neighbouring experts; only the top_groups groups with the largest score (max c, or the sum of the two largest c, of one that is left alone) take part.
// l or bias of -inf: the expert is masked, never chosen.  A place that is left over has expert -1 and weight 0.
//
// Which experts are chosen has to follow from the scores, not from how they were rounded: without a bias the order of c is that of the logits, which are
// compared as they are; with one, and where two scores of a group are added, scores are formed and compared in 64 bits.
//
// Most tokens take the short form: 16, 32 or 64 lanes share a token, at most V neighbouring experts of one group each, in registers, with the scores in 32 bits.
// A choice is a maximum over a lane's experts and over the lanes (row rotations and swaps, no LDS) and the lowest expert that has it.  Its order is that of the
// exact scores wherever neighbours in it lie further apart than both scores can be off.  Two closer sigmoid scores are compared in 64 bits by themselves; a token
// with more of them, with close groups, or with close scores of a softmax is done over with all scores in 64 bits.
// Many tokens are bound by the vector unit (8192 of 256 experts, 8 chosen: 6.5 us, with a bias 8.4, of 8 groups 9.5 to 11 by inputs), a few by the chain of choices
// (16 of them: 4 and 4.4 us).
// The long form takes tokens with a NaN, more than 256 experts, 16 groups or 16 choices, and groups too large for their lanes: with 64 lanes shared among the
// groups, as many for each as the largest power of two that they have room for, four experts a lane (240 experts in 3, 5 or 6 groups do not fit, 256 in 8 do).  A
// wavefront takes a token there, 16 experts a lane, all scores with a bias or of added pairs in 64 bits.  us, 8 chosen: 8192 tokens of 384 with a bias 47, of 1024
// 31 and with a bias 52, of 240 in 6 groups 49 and 68; 16 tokens of 384 with a bias 15, of 240 in 6 groups 25.
// The sum under the weights is of fp32 terms in the order of the lanes, of scores in 64 bits where those were formed: weights that are not divided by their own sum
// may differ in their last places with the number of tokens, and with whether theirs was done over.
#include <algorithm>
#include <type_traits>

#include "llmq_common.h"

namespace llmq {
namespace {

constexpr int kThreads = kWave, kMaxTop = 64, kMaxExperts = 1024, kMaxGroups = 64;

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

// The long form: a wavefront takes a token, V neighbouring experts each lane; the lane that has a choice notes it in LDS and looks for its next one.
template <int DT, bool EXACT, int V>
__device__ __forceinline__ void route_long(const RouteArgs& a, int64_t t) {
    constexpr int LPT = kWave;
    extern __shared__ uint64_t dyn[];  // with groups: keys of the experts, then of the groups
    __shared__ int32_t s_id[kMaxTop];
    __shared__ float s_x[kMaxTop];
    const int l = threadIdx.x, e0 = l * V;

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
        uint64_t *mine = dyn, *group = dyn + a.experts;
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

    for (int j = 0; j < a.top; j++) {
        uint64_t best = key[0];
        int bv = 0;
#pragma unroll
        for (int v = 1; v < V; v++)
            if (key[v] > best) best = key[v], bv = v;
        const uint64_t most = team_reduce<LPT>(best, [](uint64_t p, uint64_t q) { return p > q ? p : q; });
        const uint64_t have = __ballot(best == most);  // the lowest of them has the lowest expert
        if (l == __ffsll((unsigned long long)have) - 1) {
            float bx = x[0];
#pragma unroll
            for (int v = 0; v < V; v++) {
                if (v == bv) bx = x[v], key[v] = 0;
            }
            s_id[j] = most ? e0 + bv : -1;
            s_x[j] = bx;
        }
    }
    wave_fence();

    // Weights.  Renormalised ones are ratios of the chosen scores, formed relative to the largest so that none of them underflows.
    float top_x = -__builtin_inff();
    for (int j = 0; j < a.top; j++)
        if (s_id[j] >= 0) top_x = fmaxf(top_x, s_x[j]);
    auto part = [&](float v) __attribute__((always_inline)) {
        if (!a.sigmoid) return expf(v - (a.renormalize ? top_x : m));
        if (!a.renormalize || v > 0.f || top_x > 0.f) return 1.f / (1.f + expf(-v));
        return expf(v - top_x) / (1.f + expf(v));
    };
    if (a.renormalize) {
        sum = sum == sum ? 0.f : sum;  // (a softmax that has no value gives none to weights, also where the logit that took it away is not chosen)
        for (int j = 0; j < a.top; j++)
            if (s_id[j] >= 0) sum += part(s_x[j]);
    } else if (a.sigmoid) {
        sum = 1.f;
    }
    for (int j = l; j < a.top; j += LPT) {
        const int id = s_id[j];
        a.ids[t * a.top + j] = id;
        a.weights[t * a.top + j] = id < 0 ? 0.f : part(s_x[j]) / sum * a.scale;
    }
}

// ---- the short form
constexpr int kShortExperts = 256, kShortGroups = 16, kShortTop = 16;

template <int N>
__device__ __forceinline__ uint32_t rotated(uint32_t v) {  // the value N lanes on, among 16
    return (uint32_t)__builtin_amdgcn_update_dpp((int)v, (int)v, 0x120 + N, 0xf, 0xf, false);
}
template <class T, class F>  // f of the 32-bit halves of a value
__device__ __forceinline__ T by_halves(T v, F&& f) {
    if constexpr (sizeof(T) == 4) {
        return __builtin_bit_cast(T, f(__builtin_bit_cast(uint32_t, v)));
    } else {
        const uint64_t u = __builtin_bit_cast(uint64_t, v);
        return __builtin_bit_cast(T, (uint64_t)f((uint32_t)u) | (uint64_t)f((uint32_t)(u >> 32)) << 32);
    }
}
// over the LPT lanes of a token
template <int LPT, class T, class F>
__device__ __forceinline__ T over_token(T v, F&& f) {
    v = f(v, by_halves(v, [](uint32_t u) { return rotated<1>(u); })), v = f(v, by_halves(v, [](uint32_t u) { return rotated<2>(u); }));
    v = f(v, by_halves(v, [](uint32_t u) { return rotated<4>(u); })), v = f(v, by_halves(v, [](uint32_t u) { return rotated<8>(u); }));
    // (both halves of a swap of v with itself: one has the lane's own value, the other its partner's)
    if constexpr (LPT >= 32)
        v = f(by_halves(v, [](uint32_t u) { return (uint32_t)__builtin_amdgcn_permlane16_swap(u, u, false, false)[0]; }),
              by_halves(v, [](uint32_t u) { return (uint32_t)__builtin_amdgcn_permlane16_swap(u, u, false, false)[1]; }));
    if constexpr (LPT >= 64)
        v = f(by_halves(v, [](uint32_t u) { return (uint32_t)__builtin_amdgcn_permlane32_swap(u, u, false, false)[0]; }),
              by_halves(v, [](uint32_t u) { return (uint32_t)__builtin_amdgcn_permlane32_swap(u, u, false, false)[1]; }));
    return v;
}
__device__ __forceinline__ uint32_t larger(uint32_t p, uint32_t q) { return max(p, q); }
__device__ __forceinline__ float larger(float p, float q) { return fmaxf(p, q); }
__device__ __forceinline__ double larger(double p, double q) { return __builtin_fmax(p, q); }
__device__ __forceinline__ float smaller(float p, float q) { return fminf(p, q); }
__device__ __forceinline__ double smaller(double p, double q) { return __builtin_fmin(p, q); }
template <int LPT, class T>
__device__ __forceinline__ T token_max(T v) { return over_token<LPT>(v, [](T p, T q) __attribute__((always_inline)) { return larger(p, q); }); }
template <int LPT, class T>
__device__ __forceinline__ T token_sum(T v) { return over_token<LPT>(v, [](T p, T q) __attribute__((always_inline)) { return p + q; }); }
// the value of lane ^ 1, ^ 2, and of lanes that pair up where 4 or 8 neighbours agree already
template <int CTRL, class T>
__device__ __forceinline__ T paired(T v) { return by_halves(v, [](uint32_t u) { return (uint32_t)__builtin_amdgcn_mov_dpp((int)u, CTRL, 0xf, 0xf, true); }); }

__device__ __forceinline__ float exp_fast(float v) { return __builtin_amdgcn_exp2f(1.44269504088896f * v); }

// What choices go by: the logits; scores in 32 bits, where their neighbours lie far enough apart; scores in 64 bits
enum { BY_LOGITS, BY_SCORES_32, BY_SCORES_64 };

// How the experts lie: lanes_per_group lanes have a group, per_lane experts each; vec: in whole 16-byte pieces (8-byte ones in 16 bits)
struct Lay { int lanes_per_group, per_lane, vec; };

// The LPT lanes' token t, the V experts of each lane at most.  -> whether it is done, which with scores in 64 bits it is unless it has a NaN
template <int DT, int BY, int LPT, int V>
__device__ __forceinline__ bool route_short(const RouteArgs& a, Lay lay, int64_t t, bool wanted) {
    using score_t = std::conditional_t<BY == BY_SCORES_64, double, float>;
    constexpr score_t kNone = -(score_t)__builtin_inff();
    __shared__ float stage[kThreads / LPT][LPT * V];
    const int l = threadIdx.x % LPT, team = threadIdx.x / LPT, lanes_per_group = lay.lanes_per_group, per_lane = lay.per_lane;
    const uint64_t token_lanes = (LPT == 64 ? ~0ull : (1ull << (LPT & 63)) - 1) << ((threadIdx.x & (kWave - 1)) / LPT * LPT);
    const int g = l / lanes_per_group, first = l % lanes_per_group * per_lane, e0 = g * a.group_size + first;
    const int count = g < a.groups ? min(max(a.group_size - first, 0), per_lane) : 0;  // experts of the lane

    float x[V];
    if (lay.vec) {
        if constexpr (DT == LLMQ_F32) {
            const float4* p = reinterpret_cast<const float4*>((const float*)a.logits + t * a.ld + (count ? e0 : 0));
#pragma unroll
            for (int v = 0; v < V / 4; v++) {
                const float4 f = p[v];
                x[4 * v] = f.x, x[4 * v + 1] = f.y, x[4 * v + 2] = f.z, x[4 * v + 3] = f.w;
            }
        } else {
            const uint2* p = reinterpret_cast<const uint2*>((const uint16_t*)a.logits + t * a.ld + (count ? e0 : 0));
#pragma unroll
            for (int v = 0; v < V / 4; v++) {
                const uint2 f = p[v];
                x[4 * v] = Lo<DT>::lo_f32(f.x), x[4 * v + 1] = Lo<DT>::hi_f32(f.x), x[4 * v + 2] = Lo<DT>::lo_f32(f.y), x[4 * v + 3] = Lo<DT>::hi_f32(f.y);
            }
        }
    } else {
#pragma unroll
        for (int v = 0; v < V; v++) {
            const int i = l + v * LPT;
            if (i < a.experts) stage[team][i] = load_as_f32(a.logits, DT, t * a.ld + i);
        }
        wave_fence();
#pragma unroll
        for (int v = 0; v < V; v++) x[v] = v < count ? stage[team][e0 + v] : 0.f;
    }
#pragma unroll
    for (int v = 0; v < V; v++) x[v] = v < count ? x[v] : -__builtin_inff();

    float b[V];
    if constexpr (BY != BY_LOGITS) {
#pragma unroll
        for (int v = 0; v < V; v++) b[v] = 0.f;
        if (a.bias && lay.vec) {
            const float4* p = reinterpret_cast<const float4*>(a.bias + (count ? e0 : 0));
#pragma unroll
            for (int v = 0; v < V / 4; v++) {
                const float4 f = p[v];
                b[4 * v] = f.x, b[4 * v + 1] = f.y, b[4 * v + 2] = f.z, b[4 * v + 3] = f.w;
            }
        } else if (a.bias) {
#pragma unroll
            for (int v = 0; v < V; v++) b[v] = v < count ? a.bias[e0 + v] : 0.f;
        }
    }
    float m = 0.f, sum = 1.f;
    if (!a.sigmoid) {
        m = x[0];
#pragma unroll
        for (int v = 1; v < V; v++) m = fmaxf(m, x[v]);
        m = token_max<LPT>(m);
    }
    score_t key[V];  // kNone: masked, chosen already, or no expert
    score_t group = kNone, size = 0, off = 0;  // score of the lane's group and what its rounding goes by; what a score can be off, but for its last rounding
    bool sure = true;
    if constexpr (BY != BY_LOGITS) {
        score_t c[V];
        if constexpr (BY == BY_SCORES_64) {
            if (a.sigmoid) {
#pragma unroll
                for (int v = 0; v < V; v++) c[v] = 1.0 / (1.0 + exp(-(double)x[v]));
            } else {
                double all = 0.0;
#pragma unroll
                for (int v = 0; v < V; v++) c[v] = exp((double)x[v] - (double)m), all += c[v];
                // (lanes add in orders of their own; equal scores need one sum)
                static_assert(LPT == kWave, "one token");
                all = by_halves(token_sum<LPT>(all), [](uint32_t u) { return (uint32_t)__builtin_amdgcn_readfirstlane((int)u); });
                sum = (float)all;
                const double r = 1.0 / all;
#pragma unroll
                for (int v = 0; v < V; v++) c[v] *= r;
            }
        } else if (a.sigmoid) {
#pragma unroll
            for (int v = 0; v < V; v++) c[v] = __builtin_amdgcn_rcpf(1.f + exp_fast(-x[v]));
            // exp takes 2 |x| 2^-24 from its argument and 2^-23 of its own, of which s (1 - s) reaches s: less than 2^-24; the sum and the reciprocal, whose last
            // place is worth 2^-24 at most, as much each
            off = 3 * 0x1p-24f;
        } else {
            sum = 0.f;
#pragma unroll
            for (int v = 0; v < V; v++) c[v] = exp_fast(x[v] - m), sum += c[v];
            sum = token_sum<LPT>(sum);
            const float r = __builtin_amdgcn_rcpf(sum);
#pragma unroll
            for (int v = 0; v < V; v++) c[v] *= r;
            // in 2^-24 of the largest score, which is r: exp takes 2.5 d + 2 with d = m - x, of which less than 3 remain behind exp(-d); the sum's share of that
            // is at most 2.5 ln 256 + 2 < 16, which all scores have in common but the bias does not; V + 6 additions, the reciprocal 2 and the product 1
            off = (V + 32) * 0x1p-24f * r;
        }
#pragma unroll
        for (int v = 0; v < V; v++) key[v] = x[v] == -__builtin_inff() ? kNone : c[v] + (score_t)b[v];
        if (a.groups > 1) {
            score_t best = kNone, second = kNone;
#pragma unroll
            for (int v = 0; v < V; v++) second = larger(second, smaller(best, key[v])), best = larger(best, key[v]);
            auto merge = [&](score_t b2, score_t s2) __attribute__((always_inline)) {
                second = larger(smaller(best, b2), larger(second, s2));
                best = larger(best, b2);
            };
            if (lanes_per_group > 1) merge(paired<0xB1>(best), paired<0xB1>(second));   // quad_perm [1,0,3,2]
            if (lanes_per_group > 2) merge(paired<0x4E>(best), paired<0x4E>(second));   // quad_perm [2,3,0,1]
            if (lanes_per_group > 4) merge(paired<0x141>(best), paired<0x141>(second));  // row_half_mirror
            if (LPT > 16 && lanes_per_group > 8) merge(paired<0x140>(best), paired<0x140>(second));  // row_mirror
            if (LPT > 32 && lanes_per_group > 16) {
                const auto other = [&](score_t v) __attribute__((always_inline)) {  // of the 16 lanes before or behind
                    return by_halves(v, [](uint32_t u) __attribute__((always_inline)) {
                        const auto both = __builtin_amdgcn_permlane16_swap(u, u, false, false);
                        return (uint32_t)(threadIdx.x & 16 ? both[0] : both[1]);
                    });
                };
                merge(other(best), other(second));
            }
            const bool two = a.top2 && second != kNone;
            group = two ? best + second : best;
            if constexpr (BY == BY_SCORES_32) size = group == kNone ? 0.f : fabsf(best) + (two ? fabsf(second) : 0.f);
        }
    } else {
#pragma unroll
        for (int v = 0; v < V; v++) key[v] = x[v];
        if (!a.sigmoid && !a.renormalize) {
            sum = 0.f;
#pragma unroll
            for (int v = 0; v < V; v++) sum += x[v] == -__builtin_inff() ? 0.f : expf(x[v] - m);
            sum = token_sum<LPT>(sum);
        }
        if (a.groups > 1) {
            score_t best = key[0];
#pragma unroll
            for (int v = 1; v < V; v++) best = fmaxf(best, key[v]);
            if (lanes_per_group > 1) best = fmaxf(best, paired<0xB1>(best));
            if (lanes_per_group > 2) best = fmaxf(best, paired<0x4E>(best));
            if (lanes_per_group > 4) best = fmaxf(best, paired<0x141>(best));
            if (LPT > 16 && lanes_per_group > 8) best = fmaxf(best, paired<0x140>(best));
            if (LPT > 32 && lanes_per_group > 16) {
                const auto both = __builtin_amdgcn_permlane16_swap(__float_as_uint(best), __float_as_uint(best), false, false);
                best = fmaxf(__uint_as_float(both[0]), __uint_as_float(both[1]));
            }
            group = best;
        }
    }
    bool number = true;
#pragma unroll
    for (int v = 0; v < V; v += 2) number &= !__builtin_isunordered(key[v], key[v + 1]);
    sure = (__ballot(!number) & token_lanes) == 0;  // (a NaN: the long form knows its place)
    if (a.groups > 1) {
        score_t left = group, least = 0;
        // the last of as many different scores as groups are asked for, or of fewer where groups are level
        int room = a.top_groups * lanes_per_group;
        bool kept = false;
        for (int i = 0; i < a.top_groups; i++) {
            least = token_max<LPT>(left);
            const uint64_t level = __ballot(left == least) & token_lanes, below = ((uint64_t)1 << (threadIdx.x & (kWave - 1))) - 1;
            if (BY == BY_SCORES_32 && least > kNone && (int)__popcll(level) != lanes_per_group) sure = false;
            kept |= left == least && (int)__popcll(level & below) < room;  // of level ones, the lowest
            room -= (int)__popcll(level);
            left = left == least ? kNone : left;
        }
        if constexpr (BY == BY_SCORES_32) {
            const float next = token_max<LPT>(left);
            size = token_max<LPT>(size);
            // (a score and its share of the sum are each rounded once, the sum once more)
            if (least > kNone && next > kNone && !(least - next > 4 * off + 0x1p-22f * size)) sure = false;
        }
#pragma unroll
        for (int v = 0; v < V; v++) key[v] = kept ? key[v] : kNone;
    }

    // ---- the choices; lane j keeps choice j
    int id = -1;
    float before = __builtin_inff();
    bool near_last = false;  // the last two choices were close
    uint64_t pairs = 0;      // bit j: choices j - 1 and j are
    // (one choice more shows whether the last one is close to what is left, and if so one further whether those are two)
    for (int j = 0, rounds = a.top + (BY == BY_SCORES_32 ? 1 : 0); j < rounds; j++) {
        score_t best = key[0];
#pragma unroll
        for (int v = 1; v < V; v++) best = larger(best, key[v]);
        best = token_max<LPT>(best);
        int at = V;  // the lowest of the lane's experts that has it
#pragma unroll
        for (int v = V - 1; v >= 0; v--) at = key[v] == best ? v : at;
        int chosen;  // (experts lie in the order of lanes)
        if constexpr (LPT == kWave) chosen = __builtin_amdgcn_readlane(e0 + at, (__ffsll((unsigned long long)__ballot(at < V)) - 1) & (kWave - 1));
        else chosen = 0xffff - (int)token_max<LPT>(at < V ? 0xffffu - (uint32_t)(e0 + at) : 0u);
        at = chosen - e0;
#pragma unroll
        for (int v = 0; v < V; v++) key[v] = v == at ? kNone : key[v];  // (past the lane's last expert there is nothing to lose)
        if constexpr (BY == BY_SCORES_32) {
            // Two close sigmoid scores are compared in 64 bits by themselves, below; three, and those of a softmax, whose sum takes part, are not.
            const bool close = j > 0 && best > kNone && !(before - best > 2 * off + 0x1p-24f * (fabsf(before) + fabsf(best)));
            if (close && (near_last || (j <= a.top && (!a.sigmoid || j == LPT)))) sure = false;
            if (j == a.top && __any(close && sure)) rounds++;
            pairs |= (uint64_t)(close && j <= a.top) << j;
            before = best, near_last = close;
        }
        if (l == j) id = best > kNone ? chosen : -1;  // (nothing left, or nothing but NaN)
    }
    if (!__any(sure && wanted)) return false;

    float cx = id >= 0 ? load_as_f32(a.logits, DT, t * a.ld + id) : -__builtin_inff();
    if constexpr (BY == BY_SCORES_32) {
        if (__any(pairs != 0 && sure)) {
            const double score = id >= 0 ? 1.0 / (1.0 + exp(-(double)cx)) + (a.bias ? (double)a.bias[id] : 0.0) : 0.0;
            const bool second = pairs >> l & 1, first = pairs >> l >> 1 & 1;  // of its pair (no choice is in two)
            const int partner = (int)(threadIdx.x & (kWave - 1)) + (second ? -1 : first ? 1 : 0);
            auto theirs = [&](auto v) __attribute__((always_inline)) {
                return by_halves(v, [&](uint32_t u) __attribute__((always_inline)) { return (uint32_t)__builtin_amdgcn_ds_bpermute(partner * 4, (int)u); });
            };
            const double other = theirs(score);
            const int other_id = theirs(id);
            const float other_x = theirs(cx);
            const bool ahead = second ? score > other || (score == other && id < other_id) : other > score || (other == score && other_id < id);  // the second one is
            if ((first || second) && ahead) id = other_id, cx = other_x;
        }
        if (l >= a.top) id = -1, cx = -__builtin_inff();
    }

    // ---- weights, as in the long form
    const float top_x = token_max<LPT>(cx);
    float w = 0.f;
    if (id >= 0) {
        if (!a.sigmoid) w = expf(cx - (a.renormalize ? top_x : m));
        else if (!a.renormalize || cx > 0.f || top_x > 0.f) w = 1.f / (1.f + expf(-cx));
        else w = expf(cx - top_x) / (1.f + expf(cx));
    }
    if (a.renormalize) sum = token_sum<LPT>(w);
    else if (a.sigmoid) sum = 1.f;
    if (sure && wanted && l < a.top) {
        a.ids[t * a.top + l] = id;
        a.weights[t * a.top + l] = id < 0 ? 0.f : w / sum * a.scale;
    }
    return sure;
}

// Tokens that are not done at first are taken one after the other by the whole wavefront: there is one of them among thousands, and everything waits for it.  (A
// token's form depends on its own scores alone.)
template <int DT, bool EXACT, int LPT, int V>
__global__ __launch_bounds__(kThreads) void route_kernel(RouteArgs a, Lay lay, Lay alone) {
    const int64_t t0 = (int64_t)blockIdx.x * (kThreads / LPT), t = t0 + threadIdx.x / LPT;
    const bool mine = t < a.tokens;  // (lanes without a token repeat the last one's work)
    const bool done = route_short<DT, EXACT ? BY_SCORES_32 : BY_LOGITS, LPT, V>(a, lay, mine ? t : a.tokens - 1, mine);
    uint64_t left = __ballot(mine && !done);
    while (left) {
        const int lane = __ffsll((unsigned long long)left) - 1;
        const int64_t one = t0 + lane / LPT;
        left &= LPT == 64 ? 0 : ~(((1ull << (LPT & 63)) - 1) << (lane / LPT * LPT));
        if (EXACT && route_short<DT, BY_SCORES_64, kWave, kShortExperts / kWave>(a, alone, one, true)) continue;
        route_long<DT, EXACT, kShortExperts / kWave>(a, one);
    }
}
template <int DT, bool EXACT>
__global__ __launch_bounds__(kThreads) void route_many_kernel(RouteArgs a) { route_long<DT, EXACT, 16>(a, blockIdx.x); }

// -> whether LPT lanes for a token and V experts for a lane take these sizes
template <int DT, int LPT, int V>
bool lay_out(const RouteArgs& a, Lay& lay) {
    int lanes = LPT;  // of a group
    while (lanes > 1 && lanes * a.groups > LPT) lanes /= 2;
    lay.lanes_per_group = lanes, lay.per_lane = (a.group_size + lanes - 1) / lanes;
    lay.vec = a.group_size == lanes * V && a.ld % 4 == 0 && reinterpret_cast<uintptr_t>(a.logits) % (DT == LLMQ_F32 ? 16 : 8) == 0 &&
              reinterpret_cast<uintptr_t>(a.bias) % 16 == 0;
    return lanes * a.groups <= LPT && lay.per_lane <= V;
}
template <int DT, bool EXACT, int LPT, int V>
bool try_short(const RouteArgs& a, hipStream_t st) {
    Lay lay, alone;
    if (!lay_out<DT, LPT, V>(a, lay) || !lay_out<DT, kWave, kShortExperts / kWave>(a, alone)) return false;
    constexpr int kTokens = kThreads / LPT;
    hipLaunchKernelGGL((route_kernel<DT, EXACT, LPT, V>), dim3((unsigned)((a.tokens + kTokens - 1) / kTokens)), dim3(kThreads),
                       a.groups > 1 ? (a.experts + a.groups) * 8 : 0, st, a, lay, alone);
    return true;
}

// A few tokens are a chain of latencies, which fewer experts for a lane shorten; many are instructions, of which more experts for a lane need fewer.
// us without / with a bias, 16, 32, 64 lanes for a token: 16 tokens of 256 experts 5.0 4.2 3.7 / 6.0 5.1 4.5, 2048 of them 5.2 4.6 4.6 / 6.4 5.8 5.5, 8192 6.4 7.7 9.6 /
// 8.5 9.6 12.2; 16 and 32 lanes, 16 tokens of 128 4.0 3.7 / 4.8 4.5, 3000 4.2 4.5 / 5.3 5.5, 8192 4.8 6.3 / 6.0 7.9.
template <int DT, bool EXACT>
int launch_route(const RouteArgs& a, hipStream_t st) {
    bool done = false;
    if (a.groups <= kShortGroups && a.top <= kShortTop && a.experts <= kShortExperts) {
        done = try_short<DT, EXACT, 16, 4>(a, st);
        if (!done && a.tokens <= 2500) done = try_short<DT, EXACT, 32, 4>(a, st) || try_short<DT, EXACT, 64, 4>(a, st);
        if (!done) done = try_short<DT, EXACT, 16, 8>(a, st);
        if (!done && a.tokens <= 5000) done = try_short<DT, EXACT, 32, 8>(a, st);
        if (!done) done = try_short<DT, EXACT, 16, 16>(a, st);
    }
    if (!done)
        hipLaunchKernelGGL((route_many_kernel<DT, EXACT>), dim3((unsigned)a.tokens), dim3(kThreads), a.groups > 1 ? (a.experts + a.groups) * 8 : 0, st, a);
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
