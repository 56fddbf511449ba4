// fp8 quantizer with a scale per token and group of 128 channels, and the residual's addition + RMSNorm with an output in 16 or 8 bits.
//
//   group quantizer   s[m, g] = max(max_{k in g} |x[m, k]|, 1e-12) / 448        q[m, k] = e4m3(x[m, k] / s[m, g])
//   norm              h = x_dtype(x + residual)     inv = 1 / sqrt(mean_k(h^2) + eps)     y[k] = (h[k] inv) w[k]
//                     and y rounded once to x_dtype, or quantized:  int8 s = max(max_k |y|, 1e-5) / 127,  q = rint(y / s)
//                                                                   e4m3 s = max(max |y|, 1e-12) / 448, per token or per group as above
// Everything between x and the codes is fp32: sum of squares, inv, y, scales and quotients; h is what the residual stream keeps, so it is
// rounded before it is normalised.  (llmq_rmsnorm_quant_* round inv h and y to x_dtype on the way, because the reference does.)
#include <algorithm>

#include "llmq_common.h"
#include "quant_math.h"

namespace llmq {
namespace {

constexpr int kQuantThreads = 256;

// ---- group quantizer -------------------------------------------------------------------------------------------------------
// 16 lanes take a group, 16 bytes each, U groups in flight per lane; the maximum is a butterfly of lane selects.  HBM-bound: 2 bytes read, 1
// byte and 1/32 of a byte written per element.
// FLAT: rows of whole groups without gaps, so the groups are one long run and no thread divides.
template <int DT, bool FLAT, int U>
__global__ __launch_bounds__(kQuantThreads) void quant_groups_kernel(const uint16_t* __restrict__ x, int64_t ldx, int64_t K, int64_t groups,
                                                                     int64_t total, uint8_t* __restrict__ q, float* __restrict__ scale) {
    constexpr int TEAMS = kQuantThreads / kTeam;
    const int l = threadIdx.x % kTeam;
    const int64_t g0 = (int64_t)blockIdx.x * (TEAMS * U) + threadIdx.x / kTeam;
    uint4 v[U];
    int64_t at[U], to[U];  // first element of the lane's chunk in x and q; at < 0: none
    int64_t row = 0, col = 0, step_rows = 0, step_cols = 0;
    if (!FLAT) {
        row = g0 / groups, col = g0 - row * groups;
        step_rows = TEAMS / groups, step_cols = TEAMS - step_rows * groups;
    }
#pragma unroll
    for (int u = 0; u < U; u++) {
        const int64_t g = g0 + u * TEAMS;
        if (FLAT) {
            at[u] = to[u] = g < total ? g * 128 + l * 8 : -1;
        } else {
            const int64_t k = col * 128 + l * 8;
            const bool in = g < total && k < K;
            at[u] = in ? row * ldx + k : -1;
            to[u] = row * K + k;
            row += step_rows, col += step_cols;
            if (col >= groups) col -= groups, row++;
        }
        v[u] = at[u] >= 0 ? *reinterpret_cast<const uint4*>(x + at[u]) : make_uint4(0, 0, 0, 0);
    }
#pragma unroll
    for (int u = 0; u < U; u++) {
        const int64_t g = g0 + u * TEAMS;
        const float amax = team_max(absmax8(v[u], DT == LLMQ_BF16));
        const float s = scale32<MODE_F8>(amax), inv_s = 1.0f / s;
        float f[8];
        widen8<DT>(v[u], f);
        uint2 c;
        if (__all(near_ok(amax, s))) c = codes8<MODE_F8, true>(f, s, inv_s);
        else c = codes8<MODE_F8, false>(f, s, inv_s);
        if (at[u] >= 0) *reinterpret_cast<uint2*>(q + to[u]) = c;
        if (l == 0 && g < total) scale[g] = s;
    }
}

// ---- residual + RMSNorm ----------------------------------------------------------------------------------------------------
enum { OUT_SAME = LLMQ_NORM_SAME, OUT_I8 = LLMQ_NORM_I8_TOKEN, OUT_F8 = LLMQ_NORM_FP8_TOKEN, OUT_GROUP = LLMQ_NORM_FP8_GROUP };

struct NormArgs {
    const uint16_t* x;
    const uint16_t* residual;  // or null: h = x
    uint16_t* h;               // set where residual is; may be the residual itself
    const uint16_t* weight;
    uint16_t* y;               // OUT_SAME: set; otherwise optional
    uint8_t* q;
    float* scale;
    int64_t ldx, ldr, ldh, M, K;
    float eps;
};

// NT threads per row, RPB rows per block (more than one: a wavefront each, and no barrier); chunks of 8 elements tid, tid + NT, .. so that 16
// neighbours share a group.  NC > 0: a row's chunks stay in NC registers per thread between the passes; 0: rows of any length, read again.
template <int DT, int OUT, int NC, int NT, int RPB>
__global__ __launch_bounds__(NT * RPB) void add_norm_kernel(NormArgs a) {
    static_assert(RPB == 1 || NT == kWave, "several rows per block are a wavefront each");
    constexpr int MODE = OUT == OUT_I8 ? MODE_I8 : MODE_F8, REGS = NC > 0 ? NC : 1;
    __shared__ float smem[NT / kWave];
    const int tid = RPB > 1 ? threadIdx.x % kWave : threadIdx.x;
    const int64_t row = RPB > 1 ? (int64_t)blockIdx.x * RPB + threadIdx.x / kWave : blockIdx.x;
    if (RPB > 1 && row >= a.M) return;  // wavefront-uniform; no barrier follows
    const int nchunk = (int)(a.K >> 3), groups = (nchunk + kTeam - 1) / kTeam;
    const uint4* xr = reinterpret_cast<const uint4*>(a.x + row * a.ldx);
    const uint4* rr = a.residual ? reinterpret_cast<const uint4*>(a.residual + row * a.ldr) : nullptr;
    uint4* hr = a.residual ? reinterpret_cast<uint4*>(a.h + row * a.ldh) : nullptr;
    const uint4* wr = reinterpret_cast<const uint4*>(a.weight);
    uint4* yr = a.y ? reinterpret_cast<uint4*>(a.y + row * a.K) : nullptr;
    uint2* qr = reinterpret_cast<uint2*>(a.q + row * a.K);

    auto add = [&](uint4 xv, uint4 rv) __attribute__((always_inline)) {
        float f[8], g[8];
        widen8<DT>(xv, f), widen8<DT>(rv, g);
#pragma unroll
        for (int i = 0; i < 8; i++) f[i] += g[i];
        return narrow8<DT>(f);
    };
    auto sumsq = [&](uint4 v, float acc) __attribute__((always_inline)) {
        float f[8];
        widen8<DT>(v, f);
#pragma unroll
        for (int i = 0; i < 8; i++) acc = fmaf(f[i], f[i], acc);
        return acc;
    };

    uint4 hc[REGS], wc[REGS];
    float ss = 0.f;
    if (NC > 0) {
        uint4 rc[REGS];
#pragma unroll
        for (int c = 0; c < NC; c++) {
            const int i = tid + c * NT;
            hc[c] = i < nchunk ? xr[i] : make_uint4(0, 0, 0, 0);
            rc[c] = rr && i < nchunk ? rr[i] : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int c = 0; c < NC; c++) wc[c] = tid + c * NT < nchunk ? wr[tid + c * NT] : make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int c = 0; c < NC; c++) {
            if (rr) {
                hc[c] = add(hc[c], rc[c]);
                if (tid + c * NT < nchunk) hr[tid + c * NT] = hc[c];
            }
            ss = sumsq(hc[c], ss);
        }
    } else {
        for (int i = tid; i < nchunk; i += NT) {
            uint4 v = xr[i];
            if (rr) hr[i] = v = add(v, rr[i]);
            ss = sumsq(v, ss);
        }
    }
    ss = RPB > 1 ? wave_sum(ss) : block_sum<NT / kWave>(ss, smem);
    const float inv = 1.0f / sqrtf(ss / (float)a.K + a.eps);

    // h and w of chunk i; a row that is not in registers is read again, by the thread that wrote it
    auto operands = [&](int c, int i, float* h, float* w) __attribute__((always_inline)) {
        if (NC > 0) widen8<DT>(hc[c], h), widen8<DT>(wc[c], w);
        else widen8<DT>(rr ? hr[i] : xr[i], h), widen8<DT>(wr[i], w);
    };
    auto store_y = [&](int c, int i) __attribute__((always_inline)) {
        float h[8], w[8];
        operands(c, i, h, w);
#pragma unroll
        for (int e = 0; e < 8; e++) h[e] = (h[e] * inv) * w[e];
        yr[i] = narrow8<DT>(h);
    };
    // What is quantized is y / s = (h w) / (s / inv): h w is exact (two 16-bit floats), and inv, the same for scale and value, leaves the quotient, so that
    // a code depends on the rounding of s / inv = max |h w| / qmax alone.
    auto products = [&](int c, int i, float* v) __attribute__((always_inline)) {
        float w[8];
        operands(c, i, v, w);
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] *= w[e];
    };
    // scale of y, and of h w, from max |h w|
    auto scales = [&](float amax, float& s, float& sp) __attribute__((always_inline)) {
        sp = amax / QP<MODE>::qmax;
        s = sp * inv;
        if (!(amax * inv > QP<MODE>::floor_ && amax < __builtin_inff())) s = scale32<MODE>(amax * inv), sp = s / inv;  // the floor; NaN and infinity
    };
    auto each = [&](auto&& f) __attribute__((always_inline)) {  // f(register, chunk, whether it is in the row), all lanes of a wavefront together
        if (NC > 0) {
#pragma unroll
            for (int c = 0; c < NC; c++) f(c, tid + c * NT, tid + c * NT < nchunk);
        } else {
            for (int b = 0; b < nchunk; b += NT) f(0, b + tid, b + tid < nchunk);
        }
    };

    if (OUT == OUT_SAME) {
        each([&](int c, int i, bool in) __attribute__((always_inline)) {
            if (in) store_y(c, i);
        });
        return;
    }
    if (OUT == OUT_GROUP) {
        each([&](int c, int i, bool in) __attribute__((always_inline)) {
            float v[8] = {0, 0, 0, 0, 0, 0, 0, 0};
            if (in) products(c, i, v);
            float s, sp;
            const float amax = team_max(absmax8f(v));
            scales(amax, s, sp);
            const float inv_s = 1.0f / sp;
            uint2 code;
            if (__all(near_ok(amax, sp))) code = codes8<MODE, true>(v, sp, inv_s);
            else code = codes8<MODE, false>(v, sp, inv_s);
            if (!in) return;
            qr[i] = code;
            if (yr) store_y(c, i);
            if (i % kTeam == 0) a.scale[row * groups + i / kTeam] = s;
        });
        return;
    }
    float amax = 0.f;
    each([&](int c, int i, bool in) __attribute__((always_inline)) {
        if (!in) return;
        float v[8];
        products(c, i, v);
        amax = max_nonneg(amax, absmax8f(v));
        if (yr) store_y(c, i);
    });
    amax = RPB > 1 ? wave_max(amax) : block_max<NT / kWave>(amax, smem);
    float s, sp;
    scales(amax, s, sp);
    const float inv_s = 1.0f / sp;
    if (tid == 0) a.scale[row] = s;
    const bool fast = near_ok(amax, sp);  // of the row
    each([&](int c, int i, bool in) __attribute__((always_inline)) {
        if (!in) return;
        float v[8];
        products(c, i, v);
        if (fast) qr[i] = codes8<MODE, true>(v, sp, inv_s);
        else qr[i] = codes8<MODE, false>(v, sp, inv_s);
    });
}

// Threads per row and chunks per thread, by the length of a row and how many rows fill the chip: a few rows are a chain of latencies (load, reduction,
// codes), which more threads with less each shorten; many are arithmetic that every wavefront repeats per row.  A group's scale costs two
// divisions per chunk, which favours fewer chunks per thread.  us, K = 8192, 1024 x 1 / 512 x 2: 1 row int8 3.83 / 3.67, group 3.61 / 3.87; 128 rows 5.15 /
// 4.99, 5.09 / 5.36; 333 rows 7.59 / 7.20, 7.34 / 7.54.  A wavefront per row at K = 896, 8192 rows: int8 13.1 us (0.95 of a copy's rate).
template <int DT, int OUT>
int launch_add_norm(const NormArgs& a, hipStream_t st) {
    const int64_t chunks = a.K >> 3;
#define LLMQ_NORM(NC, NT, RPB) \
    hipLaunchKernelGGL((add_norm_kernel<DT, OUT, NC, NT, RPB>), dim3((unsigned)((a.M + RPB - 1) / RPB)), dim3(NT * RPB), 0, st, a)
    if (chunks <= 128 && a.M >= 256) LLMQ_NORM(2, 64, 4);
    else if (chunks <= 256) LLMQ_NORM(1, 256, 1);
    else if (chunks <= 512) {
        if (a.M < 400) LLMQ_NORM(1, 512, 1);
        else LLMQ_NORM(2, 256, 1);
    } else if (chunks <= 1024) {
        if (a.M < 400 && OUT == OUT_GROUP) LLMQ_NORM(1, 1024, 1);
        else if (a.M < 400) LLMQ_NORM(2, 512, 1);
        else LLMQ_NORM(4, 256, 1);
    } else if (chunks <= 2560) LLMQ_NORM(5, 512, 1);
    else LLMQ_NORM(0, 512, 1);
#undef LLMQ_NORM
    return launch_status();
}

template <int DT>
int add_norm_out(int out, const NormArgs& a, hipStream_t st) {
    switch (out) {
        case OUT_SAME: return launch_add_norm<DT, OUT_SAME>(a, st);
        case OUT_I8: return launch_add_norm<DT, OUT_I8>(a, st);
        case OUT_F8: return launch_add_norm<DT, OUT_F8>(a, st);
        default: return launch_add_norm<DT, OUT_GROUP>(a, st);
    }
}

template <int DT>
int launch_quant_groups(const uint16_t* x, int64_t M, int64_t K, int64_t ldx, uint8_t* q, float* scale, hipStream_t st) {
    const int64_t groups = (K + 127) / 128, total = M * groups;
    const bool flat = K % 128 == 0 && (ldx == K || M == 1);
    constexpr int TEAMS = kQuantThreads / kTeam;
#define LLMQ_QUANT(FLAT, U) \
    hipLaunchKernelGGL((quant_groups_kernel<DT, FLAT, U>), dim3((unsigned)((total + TEAMS * U - 1) / (TEAMS * U))), dim3(kQuantThreads), 0, st, \
                       x, ldx, K, groups, total, q, scale)
    if (total >= 256 * TEAMS * 8) {
        if (flat) LLMQ_QUANT(true, 4);
        else LLMQ_QUANT(false, 4);
    } else {
        if (flat) LLMQ_QUANT(true, 1);
        else LLMQ_QUANT(false, 1);
    }
#undef LLMQ_QUANT
    return launch_status();
}

bool aligned8(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 7u) == 0; }

}  // namespace
}  // namespace llmq

using namespace llmq;

extern "C" int llmq_quant_fp8_per_group(const void* x, int x_dtype, int64_t M, int64_t K, int64_t ldx, uint8_t* q, float* scale,
                                        llmq_stream_t stream) {
    if (x_dtype != LLMQ_BF16 && x_dtype != LLMQ_F16) return LLMQ_ERR_DTYPE;
    if (M < 0 || K < 0 || M > 0x7fffffffLL || K > 0x7fffffffLL || ldx < K || (K & 7) || (ldx & 7)) return LLMQ_ERR_SHAPE;
    if (M == 0 || K == 0) return LLMQ_OK;
    if (!x || !q || !scale) return LLMQ_ERR_NULL;
    if (!aligned16(x) || !aligned8(q)) return LLMQ_ERR_ALIGN;
    // a grid holds fewer than 2^32 threads: rows beyond that many go to further launches
    const int64_t groups = (K + 127) / 128, step = std::max<int64_t>(1, ((int64_t)1 << 27) / groups);
    int rc = LLMQ_OK;
    for (int64_t m = 0; m < M && rc == LLMQ_OK; m += step) {
        const uint16_t* xm = (const uint16_t*)x + m * ldx;
        const int64_t rows = std::min(step, M - m);
        rc = x_dtype == LLMQ_BF16 ? launch_quant_groups<LLMQ_BF16>(xm, rows, K, ldx, q + m * K, scale + m * groups, (hipStream_t)stream)
                                  : launch_quant_groups<LLMQ_F16>(xm, rows, K, ldx, q + m * K, scale + m * groups, (hipStream_t)stream);
    }
    return rc;
}

extern "C" int llmq_add_rmsnorm(int out, const void* x, int x_dtype, int64_t M, int64_t K, int64_t ldx, const void* residual, int64_t ldr,
                                void* h, int64_t ldh, const void* weight, float eps, void* y, void* q, float* scale, llmq_stream_t stream) {
    if (out < OUT_SAME || out > OUT_GROUP || (x_dtype != LLMQ_BF16 && x_dtype != LLMQ_F16)) return LLMQ_ERR_DTYPE;
    if (M < 0 || K < 0 || M > 0x7fffffffLL || K > 0x7fffffffLL || ldx < K || (K & 7) || (ldx & 7)) return LLMQ_ERR_SHAPE;
    if (residual && (ldr < K || ldh < K || (ldr & 7) || (ldh & 7))) return LLMQ_ERR_SHAPE;
    if (M == 0) return LLMQ_OK;
    if (K == 0) return LLMQ_ERR_SHAPE;
    if (!x || !weight || (residual && !h) || (out == OUT_SAME ? !y : (!q || !scale))) return LLMQ_ERR_NULL;
    if (!aligned16(x) || !aligned16(weight) || (residual && (!aligned16(residual) || !aligned16(h))) || (y && !aligned16(y)) ||
        (out != OUT_SAME && !aligned8(q)))
        return LLMQ_ERR_ALIGN;
    const int64_t per_row = out == OUT_GROUP ? (K + 127) / 128 : 1, step = (int64_t)1 << 21;  // rows of a grid: 2^32 threads are too many
    int rc = LLMQ_OK;
    for (int64_t m = 0; m < M && rc == LLMQ_OK; m += step) {
        NormArgs a = {};
        a.x = (const uint16_t*)x + m * ldx, a.weight = (const uint16_t*)weight;
        if (residual) a.residual = (const uint16_t*)residual + m * ldr, a.h = (uint16_t*)h + m * ldh;
        if (y) a.y = (uint16_t*)y + m * K;
        if (out != OUT_SAME) a.q = (uint8_t*)q + m * K, a.scale = scale + m * per_row;
        a.ldx = ldx, a.ldr = ldr, a.ldh = ldh, a.M = std::min(step, M - m), a.K = K, a.eps = eps;
        rc = x_dtype == LLMQ_BF16 ? add_norm_out<LLMQ_BF16>(out, a, (hipStream_t)stream) : add_norm_out<LLMQ_F16>(out, a, (hipStream_t)stream);
    }
    return rc;
}
