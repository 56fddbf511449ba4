// Block-scaled fp8 product for up to 64 tokens: weight rows streamed through LDS in long pieces.
//
//   out[m, n] = sum_b sa[m, b] sw[n / 128, b] sum_{k in block b} A[m, k] B[n, k]   (+ bias[n])
//
// Bound by the stream of weights out of HBM.  A block of four wavefronts owns 16 T channels and 16 MT tokens over the whole K.  A stage is SEG =
// 512 STEPS bytes of K of every weight and activation row, loaded straight into LDS, NS - 1 stages in flight beside the one that is
// multiplied; each wavefront takes STEPS blocks of 128 of a stage, one MFMA each, and scales the results into its own fp32 sums with the scales that
// it loaded with the stage.  The four sums are added in wavefront order at the end: no K split, no second launch, a fixed order.
// MANY: for many channels as many blocks as are resident take one group of 16 T channels after the other; the ring runs on into the next group while the
// last one's sums are added beside it.
#include <algorithm>
#include <type_traits>

#include "gemm_block.h"

namespace llmq {
namespace {

typedef int v8i __attribute__((ext_vector_type(8)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));

constexpr int kMostGroups = 16;  // groups of channels that a block takes

template <int T_, int MT_, int STEPS_, int NS_, bool MANY_>
struct RowsCfg {
    static constexpr int T = T_, MT = MT_, STEPS = STEPS_, NS = NS_;
    static constexpr bool MANY = MANY_;
    static constexpr int NW = 4, NT = NW * kWave, SEG = 512 * STEPS, CPR = SEG / 16;
    static constexpr int ROWS = 16 * (T + MT), DATA = ROWS * SEG;
    static constexpr int SLOADS = 16 * MT + 1 > kWave ? 2 : 1, SWAVE = STEPS * SLOADS * kWave * 4;  // scale loads per block of K; bytes of a wavefront's
    static constexpr int STAGE = DATA + NW * SWAVE, LPT = DATA / (NT * 16), LOADS = LPT + STEPS * SLOADS;
    static constexpr int RING = NS * STAGE, SUMS = NW * T * MT * kWave * 16;
    static constexpr int BIAS = (MANY ? kMostGroups : 1) * 16 * T * 4;
    static constexpr int LDS_BYTES = (MANY ? RING + SUMS : (RING > SUMS ? RING : SUMS)) + BIAS;
    static_assert(DATA % (NT * 16) == 0 && LDS_BYTES <= 160 * 1024 && (NS - 1) * LOADS < 64 && 128 % (16 * T) == 0, "even stages, LDS, vmcnt, one block of channels");
};

template <class C>
__global__ __launch_bounds__(C::NT) void block_rows_kernel(BlockArgs g) {
    extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
    constexpr int T = C::T, MT = C::MT, NS = C::NS, SEG = C::SEG;
    const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(tid / kWave);
    const int l16 = lane & 15, kq = lane >> 4;
    int n0 = blockIdx.x * (16 * T);
    const int nst = (g.K + SEG - 1) / SEG, step_n = C::MANY ? gridDim.x * (16 * T) : 0;
    const int groups = C::MANY ? (g.N - 1 - n0) / max(step_n, 1) + 1 : 1, total = groups * nst;  // of channels; stages of the block

    // ---- direct loads: piece p of a stage is row p / CPR (weights, then activations), LDS chunk p % CPR, which holds chunk (p % CPR) ^ (row & 15)
    // of the row, so that the operand reads of 16 rows hit 16 places; rows past the end are the last one again
    uint32_t off[C::LPT], chunk[C::LPT];
    const uint8_t* b_base;
    const float *sa_row, *sw_row;
    auto aim = [&](int n) __attribute__((always_inline)) {  // the loads of a group
        b_base = g.B + (int64_t)n * g.ldb;
#pragma unroll
        for (int i = 0; i < C::LPT; i++) {
            const int row = ((wave * C::LPT + i) * kWave + lane) / C::CPR;
            off[i] = row < 16 * T ? (uint32_t)min(row, g.N - 1 - n) * (uint32_t)g.ldb : (uint32_t)min(row - 16 * T, g.M - 1) * (uint32_t)g.lda;
        }
        sw_row = g.sw + (int64_t)(n / kScaleBlock) * g.KB;
        sa_row = lane < 16 * MT ? g.sa + (int64_t)min(lane, g.M - 1) * g.KB : sw_row;  // the lane behind the tokens fetches the weights' scale
    };
#pragma unroll
    for (int i = 0; i < C::LPT; i++) {
        const int p = (wave * C::LPT + i) * kWave + lane;
        chunk[i] = 16u * (uint32_t)((p % C::CPR) ^ ((p / C::CPR) & 15));
    }
    aim(n0);
    const uint32_t lds_base = (uint32_t)(uintptr_t)((__attribute__((address_space(3))) void*)smem);
    auto issue = [&](int s, int slot) __attribute__((always_inline)) {
        const bool tail = (s + 1) * SEG > g.K;  // uniform: chunks past the end re-read the last one of the row, masked when used
        const uint32_t to = lds_base + (uint32_t)slot * C::STAGE;
#pragma unroll
        for (int i = 0; i < C::LPT; i++) {
            const bool w = (wave * C::LPT + i) * kWave < 16 * T * C::CPR;  // wavefront-uniform
            const uint8_t* src = (w ? b_base : g.A) + (int64_t)s * SEG;
            uint32_t voff = off[i] + chunk[i];
            if (tail) voff = off[i] + min(chunk[i], (uint32_t)(g.K - 16 - s * SEG));
            const uint32_t m0v = to + (uint32_t)(wave * C::LPT + i) * 1024;
            asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(m0v), "v"(voff), "s"(src) : "memory", "m0");
        }
#pragma unroll
        for (int step = 0; step < C::STEPS; step++) {
            const int kb = min((s * C::NW + wave) * C::STEPS + step, g.KB - 1);
#pragma unroll
            for (int k = 0; k < C::SLOADS; k++) {
                const float* p = (k ? sw_row : sa_row) + kb;
                const uint32_t m0v = to + C::DATA + (uint32_t)wave * C::SWAVE + (uint32_t)(step * C::SLOADS + k) * (kWave * 4);
                asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off" ::"s"(m0v), "v"(p) : "memory", "m0");
            }
        }
    };
    auto lds_barrier = []() __attribute__((always_inline)) {  // orders LDS traffic only: the loads stay in flight across it
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
    };

    v4f acc[MT][T];
    auto clear = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (int mt = 0; mt < MT; mt++)
#pragma unroll
            for (int t = 0; t < T; t++) acc[mt][t] = v4f{0, 0, 0, 0};
    };
    clear();
    auto read = [&](const uint8_t* st, int row, int step, bool tail, int left) __attribute__((always_inline)) {
        const u4* r = reinterpret_cast<const u4*>(st + row * SEG);
        const int c = (wave * C::STEPS + step) * 8 + 2 * kq;
        u4 lo = r[c ^ l16], hi = r[(c + 1) ^ l16];
        if (tail) {
            if (16 * c >= left) lo = u4{0, 0, 0, 0};
            if (16 * (c + 1) >= left) hi = u4{0, 0, 0, 0};
        }
        return v8i{(int)lo[0], (int)lo[1], (int)lo[2], (int)lo[3], (int)hi[0], (int)hi[1], (int)hi[2], (int)hi[3]};
    };
    auto compute = [&](int slot, bool tail, int left) __attribute__((always_inline)) {
        const uint8_t* st = smem + slot * C::STAGE;
#pragma unroll
        for (int step = 0; step < C::STEPS; step++) {
            if (tail && (wave * C::STEPS + step) * kScaleBlock >= left) continue;  // no block (the scales loaded for it are the last one's); wavefront-uniform
            const float* sc = reinterpret_cast<const float*>(st + C::DATA + wave * C::SWAVE + step * C::SLOADS * kWave * 4);
            v8i b[T], a[MT];
#pragma unroll
            for (int t = 0; t < T; t++) b[t] = read(st, 16 * t + l16, step, tail, left);
#pragma unroll
            for (int mt = 0; mt < MT; mt++) a[mt] = read(st, 16 * (T + mt) + l16, step, tail, left);
            const float w = sc[16 * MT];
#pragma unroll
            for (int mt = 0; mt < MT; mt++) {
                const float f = sc[16 * mt + l16] * w;
                v4f p[T];
#pragma unroll
                for (int t = 0; t < T; t++) p[t] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(b[t], a[mt], v4f{0, 0, 0, 0}, 0, 0, 0, 0, 0, 0);
#pragma unroll
                for (int t = 0; t < T; t++)
#pragma unroll
                    for (int e = 0; e < 4; e++) acc[mt][t][e] = fmaf(p[t][e], f, acc[mt][t][e]);
            }
        }
    };
    auto wait_stage = [&](int younger) __attribute__((always_inline)) {  // the oldest stage in flight has landed when `younger` later ones remain
        if (NS > 3 && younger == 2) { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(NS > 3 ? 2 * C::LOADS : 0) : "memory"); return; }
        if (NS > 2 && younger == 1) { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(NS > 2 ? C::LOADS : 0) : "memory"); return; }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    };
    static_assert(NS <= 4, "wait_stage");

    // the bias of all the block's channels waits in LDS: a load at the end of a group would wait behind the ring
    float* s_bias = reinterpret_cast<float*>(smem + C::LDS_BYTES - C::BIAS);
    if (g.bias) {
        for (int i = tid; i < groups * 16 * T; i += C::NT)
            s_bias[i] = load_as_f32(g.bias, g.bias_dtype, min(n0 + i / (16 * T) * step_n + i % (16 * T), g.N - 1));
    }
    v4f (*red)[MT * T][kWave] = reinterpret_cast<v4f (*)[MT * T][kWave]>(smem + (C::MANY ? C::RING : 0));
    auto finish = [&](int group) __attribute__((always_inline)) {
#pragma unroll
        for (int mt = 0; mt < MT; mt++)
#pragma unroll
            for (int t = 0; t < T; t++) red[wave][mt * T + t][lane] = acc[mt][t];
        lds_barrier();
        for (int idx = tid; idx < MT * T * kWave; idx += C::NT) {
            const int q = idx / kWave, l = idx % kWave, mt = q / T, t = q % T;
            v4f sum = red[0][q][l];
#pragma unroll
            for (int w = 1; w < C::NW; w++) sum += red[w][q][l];
            // lane l: token 16 mt + l % 16, channels 16 t + 4 (l / 16) .. + 3
            const int m = 16 * mt + (l & 15), c = 16 * t + 4 * (l >> 4), n = n0 + c;
            if (m >= g.M || n >= g.N) continue;
            uint16_t h[4];
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const float v = sum[e] + (g.bias ? s_bias[group * 16 * T + c + e] : 0.f);
                h[e] = g.out_dtype == LLMQ_BF16 ? Lo<LLMQ_BF16>::from_f32(v) : Lo<LLMQ_F16>::from_f32(v);
            }
            uint16_t* to = reinterpret_cast<uint16_t*>(g.out) + (int64_t)m * g.ldo + n;
            typedef uint32_t u2v __attribute__((ext_vector_type(2)));
            typedef u2v u2any __attribute__((aligned(2)));  // (rows of an odd number of channels start at any even address)
            if (n + 3 < g.N)
                *reinterpret_cast<u2any*>(to) = u2v{(uint32_t)h[0] | ((uint32_t)h[1] << 16), (uint32_t)h[2] | ((uint32_t)h[3] << 16)};
            else
#pragma unroll
                for (int e = 0; e < 4; e++)
                    if (n + e < g.N) to[e] = h[e];
        }
    };

    int issued = 0, issue_s = 0, issue_n = n0;  // stages requested; the next one within its group
    auto issue_next = [&](int slot) __attribute__((always_inline)) {
        if (issued == total) return;
        if (C::MANY && issue_s == nst) issue_s = 0, issue_n += step_n, aim(issue_n);
        issue(issue_s++, slot);
        issued++;
    };
#pragma unroll
    for (int t = 0; t < NS - 1; t++) issue_next(t);
    int slot = 0, s = 0, group = 0;
#pragma unroll 1
    for (int f = 0; f < total; f++) {
        wait_stage(min(total - 1, f + NS - 2) - f);
        lds_barrier();  // publishes this stage; every wavefront has read the whole of the one before
        issue_next(slot == 0 ? NS - 1 : slot - 1);
        if ((s + 1) * SEG > g.K) compute(slot, true, g.K - s * SEG);
        else compute(slot, false, 0);
        slot = slot == NS - 1 ? 0 : slot + 1;
        s++;
        if (C::MANY && s == nst) {
            finish(group);  // its reads of the sums are done in every wavefront before the barrier of the next stage
            clear();
            group++, s = 0;
            if (group < groups) n0 += step_n;
        }
    }
    if constexpr (!C::MANY) {
        lds_barrier();  // every wavefront is done reading the stages
        finish(0);
    }
}

template <class C>
int launch_rows(const BlockArgs& g, hipStream_t st) {
    auto kernel = block_rows_kernel<C>;
    if (C::LDS_BYTES > 64 * 1024) {
        static bool raised[64] = {};  // per device: the attribute belongs to the loaded code object of the current device
        int dev = 0;
        if (hipGetDevice(&dev) != hipSuccess) return LLMQ_ERR_LAUNCH;
        if (dev < 0 || dev >= 64 || !raised[dev]) {
            if (hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, C::LDS_BYTES) != hipSuccess)
                return LLMQ_ERR_LAUNCH;
            if (dev >= 0 && dev < 64) raised[dev] = true;
        }
    }
    int64_t blocks = ((int64_t)g.N + 16 * C::T - 1) / (16 * C::T);
    if (C::MANY) {  // as many as are resident at once, or fewer so that all take as many groups
        const int64_t slots = 256 * (160 * 1024 / C::LDS_BYTES), each = std::min<int64_t>(kMostGroups, (blocks + slots - 1) / slots);
        blocks = (blocks + each - 1) / each;
    }
    if (blocks * C::NT > 0xffffffffLL) return LLMQ_ERR_SHAPE;
    hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(C::NT), C::LDS_BYTES, st, g);
    return launch_status();
}

}  // namespace

int launch_block_rows(int variant, const BlockArgs& g, hipStream_t st) {
    switch (variant) {
#define LLMQ_BLOCK_ROWS_CASE(I, T, MT, STEPS, NS, MANY) \
    case I: return launch_rows<RowsCfg<T, MT, STEPS, NS, MANY>>(g, st);
        LLMQ_BLOCK_ROWS(LLMQ_BLOCK_ROWS_CASE)
#undef LLMQ_BLOCK_ROWS_CASE
    }
    return LLMQ_ERR_SHAPE;
}

}  // namespace llmq
