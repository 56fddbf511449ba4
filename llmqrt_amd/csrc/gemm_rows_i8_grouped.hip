// W8A8 product by experts, a few rows each: weight rows streamed through LDS in long pieces.
//
//   out[m, n] = dtype( (acc[m, n] a_scale[m]) w_scale[e, n] + bias[e, n] ),  acc[m, n] = sum_k A[m, k] B[e, n, k],  m of expert e
//
// Bound by the stream of weights out of HBM.  A block of four wavefronts takes 16 T channels and 16 MT rows of one expert over the whole K, then its
// next such item: as many blocks as are resident share the items, and the ring of stages runs on from one item into the next, so that a CU is
// never without loads.  A stage is 512 bytes of K of every weight and activation row, straight into LDS, with the item's scales and bias beside
// it; each wavefront multiplies a quarter of it, and the four sums are added at the end of an item.  Sums are whole numbers: any order gives the same.
// 32 channels and 3 stages, 16 channels and 4, tiles of 32 x 128 and 64 x 128, us: 48 rows of 64 experts, 2048 x 2048, 26.8 33.2 28.3 28.9; 256 rows of them (268 MB of
// weights, 5.4 TB/s) 49.4 58.8 47.5 50; 8 rows of 8, 4864 x 3584, 17.0 19.9 17.6 18.3.
#include <algorithm>

#include "expert_tiles.h"
#include "gemm_grouped.h"

namespace llmq {
namespace {

typedef int v4i __attribute__((ext_vector_type(4)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));

template <int T_, int MT_, int NS_>
struct GRowsCfg {
    static constexpr int T = T_, MT = MT_, NS = NS_;
    static constexpr int SEG = 512, NW = 4, NT = NW * kWave, CPR = SEG / 16, STEPS = SEG / NW / 64;
    static constexpr int ROWS = 16 * (T + MT), DATA = ROWS * SEG, SCALES = NW * kWave * 4 + 16;  // channels' scales, rows' scales, bias, the item
    static constexpr int STAGE = DATA + SCALES, LPT = DATA / (NT * 16), LOADS = LPT + 1;
    static constexpr int TABLE = (2 * kGroupedRowsExperts + 1) * 4;
    static constexpr int LDS_BYTES = NS * STAGE + (TABLE + 15) / 16 * 16;
    static_assert(DATA % (NT * 16) == 0 && LDS_BYTES <= 160 * 1024 && (NS - 1) * LOADS < 64 && 16 * T <= kWave && 16 * MT <= kWave, "even stages, LDS, vmcnt");
    static_assert(NW * T * MT * kWave * 16 <= DATA && STAGE % 16 == 0, "the wavefronts' sums take a stage's place");
};

template <class C>
__global__ __launch_bounds__(C::NT) void grouped_rows_kernel(GroupedCall g) {
    extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
    constexpr int T = C::T, MT = C::MT, NS = C::NS, SEG = C::SEG;
    const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(tid / kWave);
    const int r16 = lane & 15, kq = lane >> 4;
    const int nst = (g.K + SEG - 1) / SEG, tiles_n = (g.N + 16 * T - 1) / (16 * T);

    // ---- the experts' first rows and their slabs of 16 MT rows, counted up: offsets as in expert_tile
    int32_t* s_upto = reinterpret_cast<int32_t*>(smem + NS * C::STAGE);  // slabs of experts 0 .. e
    int32_t* s_first = s_upto + kGroupedRowsExperts;
    if (wave == 0) {
        int from = 0, total = 0;
        for (int e0 = 0; e0 < g.experts; e0 += kWave) {
            const bool in = e0 + lane < g.experts;  // (the lane behind the last expert has its end)
            const int first = max(from, wave_prefix_max(e0 + lane <= g.experts ? min(max(g.offsets[e0 + lane], 0), g.M) : 0));
            const int last = in ? max(first, min(g.offsets[e0 + lane + 1], g.M)) : first;
            const int upto = total + wave_prefix((last - first + 16 * MT - 1) / (16 * MT));
            if (in) s_upto[e0 + lane] = upto, s_first[e0 + lane] = first;
            from = __builtin_amdgcn_readlane(last, kWave - 1), total = __builtin_amdgcn_readlane(upto, kWave - 1);
        }
        if (lane == 0) s_first[g.experts] = from;
    }
    __syncthreads();

    // ---- the block's items: every XCD has a range of them, so that slabs with the same weights meet in one L2
    const int items = __builtin_amdgcn_readfirstlane(s_upto[g.experts - 1]) * tiles_n;
    const int xcd = blockIdx.x % kExpertXcd, per = gridDim.x / kExpertXcd;
    const int lo = (int)((int64_t)items * xcd / kExpertXcd), hi = (int)((int64_t)items * (xcd + 1) / kExpertXcd);
    int item = lo + (int)(blockIdx.x / kExpertXcd);  // the next one to load
    if (item >= hi) return;  // block-uniform
    const int total = ((hi - item + per - 1) / per) * nst;  // stages

    // ---- direct loads: piece p of a stage is row p / CPR (weights, then activations), LDS chunk p % CPR, which holds chunk (p % CPR) ^ (row & 15)
    // of the row, so that the operand reads of 16 rows hit 16 places; rows past the end are the last one again
    const uint8_t *a_base, *b_base, *extra;  // extra: this lane's element of the wavefront's scales or bias
    uint32_t off[C::LPT], chunk[C::LPT];
    int n0, row0, rows, look = 0;  // of the item that is loaded
    const bool bias16 = g.ep.bias && g.ep.bias_dtype != LLMQ_F32;
    auto aim = [&]() __attribute__((always_inline)) {
        const int slab = item / tiles_n;
        int e, before;
        while (true) {  // 64 experts at a time; the items only go up
            const int at = look + lane;
            const uint64_t has = __ballot(at < g.experts && slab < s_upto[min(at, g.experts - 1)]);
            if (has) {
                e = look + __ffsll((unsigned long long)has) - 1;
                break;
            }
            look += kWave;
        }
        e = __builtin_amdgcn_readfirstlane(e);
        before = __builtin_amdgcn_readfirstlane(e ? s_upto[e - 1] : 0);
        const int slabs = __builtin_amdgcn_readfirstlane(s_upto[e]) - before, rest = item - before * tiles_n;
        const int tn = rest / slabs, first = __builtin_amdgcn_readfirstlane(s_first[e]), last = __builtin_amdgcn_readfirstlane(s_first[e + 1]);
        n0 = tn * (16 * T);
        row0 = first + (rest - tn * slabs) * (16 * MT);
        rows = min(last - row0, 16 * MT);
        a_base = g.A + (int64_t)row0 * g.lda;
        b_base = g.B + ((int64_t)e * g.N + n0) * g.K;
        const int64_t channel = (int64_t)e * g.N + min(n0 + min(lane, 16 * T - 1), g.N - 1);
        const float* scale = wave == 1 ? g.ep.a_scale + row0 + min(lane, rows - 1) : g.ep.w_scale + channel;
        extra = reinterpret_cast<const uint8_t*>(scale);
        if (wave == 2 && g.ep.bias) extra = (const uint8_t*)g.ep.bias + channel * (bias16 ? 2 : 4);
#pragma unroll
        for (int i = 0; i < C::LPT; i++) {
            const int row = ((wave * C::LPT + i) * kWave + lane) / C::CPR;
            off[i] = row < 16 * T ? (uint32_t)min(row, g.N - 1 - n0) * (uint32_t)g.K : (uint32_t)min(row - 16 * T, rows - 1) * (uint32_t)g.lda;
        }
    };
#pragma unroll
    for (int i = 0; i < C::LPT; i++) {
        const int p = (wave * C::LPT + i) * kWave + lane;
        chunk[i] = 16u * (uint32_t)((p % C::CPR) ^ ((p / C::CPR) & 15));
    }
    const uint32_t lds_base = (uint32_t)(uintptr_t)((__attribute__((address_space(3))) void*)smem);
    auto issue = [&](int s, int slot) __attribute__((always_inline)) {
        const bool tail = (s + 1) * SEG > g.K;  // uniform: chunks past the end re-read the last one of the row, masked when used
        const uint32_t to = lds_base + (uint32_t)slot * C::STAGE;
#pragma unroll
        for (int i = 0; i < C::LPT; i++) {
            const bool w = (wave * C::LPT + i) * kWave < 16 * T * C::CPR;  // wavefront-uniform
            const uint8_t* src = (w ? b_base : a_base) + (int64_t)s * SEG;
            uint32_t voff = off[i] + chunk[i];
            if (tail) voff = off[i] + min(chunk[i], (uint32_t)(g.K - 16 - s * SEG));
            const uint32_t m0v = to + (uint32_t)(wave * C::LPT + i) * 1024;
            asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(m0v), "v"(voff), "s"(src) : "memory", "m0");
        }
        const uint32_t m0v = to + C::DATA + (uint32_t)wave * (kWave * 4);
        if (wave == 2 && bias16) asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_ushort %1, off" ::"s"(m0v), "v"(extra) : "memory", "m0");
        else asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off" ::"s"(m0v), "v"(extra) : "memory", "m0");
        if (tid == 0) *reinterpret_cast<int4*>(smem + slot * C::STAGE + C::DATA + C::NW * kWave * 4) = make_int4(n0, row0, rows, 0);
    };
    auto lds_barrier = []() __attribute__((always_inline)) {  // orders LDS traffic only: the loads stay in flight across it
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
    };

    v4i acc[MT][T];
    auto clear = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (int mt = 0; mt < MT; mt++)
#pragma unroll
            for (int t = 0; t < T; t++) acc[mt][t] = v4i{0, 0, 0, 0};
    };
    clear();
    auto read = [&](const uint8_t* st, int row, int step, bool tail, int left) __attribute__((always_inline)) {  // row of the stage
        const int c = (wave * C::STEPS + step) * 4 + kq;
        u4 v = reinterpret_cast<const u4*>(st + row * SEG)[c ^ r16];
        if (tail && 16 * c >= left) v = u4{0, 0, 0, 0};
        return v4i{(int)v[0], (int)v[1], (int)v[2], (int)v[3]};
    };
    auto compute = [&](const uint8_t* st, bool tail, int left) __attribute__((always_inline)) {
#pragma unroll
        for (int step = 0; step < C::STEPS; step++) {
            v4i b[T], a[MT];
#pragma unroll
            for (int t = 0; t < T; t++) b[t] = read(st, 16 * t + r16, step, tail, left);
#pragma unroll
            for (int mt = 0; mt < MT; mt++) a[mt] = read(st, 16 * (T + mt) + r16, step, tail, left);
#pragma unroll
            for (int mt = 0; mt < MT; mt++)
#pragma unroll
                for (int t = 0; t < T; t++) acc[mt][t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(b[t], a[mt], acc[mt][t], 0, 0, 0);
        }
    };
    auto wait_stage = [&](int younger) __attribute__((always_inline)) {  // the oldest stage in flight has landed when `younger` later ones remain
        if (NS > 3 && younger == 2) { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(NS > 3 ? 2 * C::LOADS : 0) : "memory"); return; }
        if (NS > 2 && younger == 1) { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(NS > 2 ? C::LOADS : 0) : "memory"); return; }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    };
    static_assert(NS <= 4, "wait_stage");

    // the end of an item, in the stage of its last loads
    auto finish = [&](uint8_t* st) __attribute__((always_inline)) {
        v4i (*red)[MT * T][kWave] = reinterpret_cast<v4i (*)[MT * T][kWave]>(st);
        lds_barrier();  // every wavefront has read its operands
#pragma unroll
        for (int mt = 0; mt < MT; mt++)
#pragma unroll
            for (int t = 0; t < T; t++) red[wave][mt * T + t][lane] = acc[mt][t];
        lds_barrier();
        const float *s_w = reinterpret_cast<const float*>(st + C::DATA), *s_a = s_w + kWave, *s_b = s_a + kWave;
        const int4 at = *reinterpret_cast<const int4*>(s_w + C::NW * kWave);  // first channel, first row, rows
        for (int idx = tid; idx < MT * T * kWave; idx += C::NT) {
            const int q = idx / kWave, l = idx % kWave, mt = q / T, t = q % T;
            v4i sum = red[0][q][l];
#pragma unroll
            for (int w = 1; w < C::NW; w++) sum += red[w][q][l];
            // lane l of that accumulator: row 16 mt + l % 16, channels 16 t + 4 (l / 16) .. + 3
            const int m = 16 * mt + (l & 15), c = 16 * t + 4 * (l >> 4), n = at.x + c;
            if (m >= at.z || n >= g.N) continue;
            const float sa = s_a[m];
            uint16_t h[4];
#pragma unroll
            for (int e = 0; e < 4; e++) {
                float bb = s_b[c + e];
                if (bias16) bb = g.ep.bias_dtype == LLMQ_BF16 ? Lo<LLMQ_BF16>::to_f32((uint16_t)__float_as_uint(bb)) : Lo<LLMQ_F16>::to_f32((uint16_t)__float_as_uint(bb));
                const float v = g.ep.bias ? epi_value<false>((float)sum[e], sa, s_w[c + e], 1.f, bb) : epi_value<true>((float)sum[e], sa, s_w[c + e], 1.f, 0.f);
                h[e] = g.ep.out_dtype == LLMQ_BF16 ? Lo<LLMQ_BF16>::from_f32(v) : Lo<LLMQ_F16>::from_f32(v);
            }
            uint16_t* to = reinterpret_cast<uint16_t*>(g.out) + (int64_t)(at.y + m) * g.ldo + n;
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

    int issued = 0, issue_s = 0;  // stages requested; the next one within its item
    aim();
    auto issue_next = [&](int slot) __attribute__((always_inline)) {
        if (issued == total) return;
        if (issue_s == nst) issue_s = 0, item += per, aim();
        issue(issue_s++, slot);
        issued++;
    };
#pragma unroll
    for (int t = 0; t < NS - 1; t++) issue_next(t);
    int slot = 0, s = 0;
#pragma unroll 1
    for (int f = 0; f < total; f++) {
        wait_stage(min(total - 1, f + NS - 2) - f);
        lds_barrier();  // publishes this stage; every wavefront is done with the whole of the one before
        issue_next(slot == 0 ? NS - 1 : slot - 1);
        uint8_t* st = smem + slot * C::STAGE;
        if ((s + 1) * SEG > g.K) compute(st, true, g.K - s * SEG);
        else compute(st, false, 0);
        slot = slot == NS - 1 ? 0 : slot + 1;
        if (++s == nst) {
            finish(st);
            clear();
            s = 0;
        }
    }
}

template <class C, int PER_CU>
int launch_rows(const GroupedCall& g, hipStream_t st) {
    auto kernel = grouped_rows_kernel<C>;
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
    const int64_t slabs = g.M / (16 * C::MT) + std::min(g.experts, g.M), items = slabs * cdiv(g.N, 16 * C::T);
    if (items > 0x7fffffffLL || g.experts > kGroupedRowsExperts) return LLMQ_ERR_SHAPE;
    static_assert(PER_CU == 160 * 1024 / C::LDS_BYTES, "resident blocks");
    const int64_t slots = 256 * PER_CU, blocks = (std::min(items, slots) + kExpertXcd - 1) / kExpertXcd * kExpertXcd;
    hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(C::NT), C::LDS_BYTES, st, g);
    return launch_status();
}

}  // namespace

int launch_grouped_rows(int variant, const GroupedCall& g, hipStream_t st) {
    switch (variant) {
#define LLMQ_GROUPED_ROWS_CASE(I, T, MT, NS, CU) \
    case I: return launch_rows<GRowsCfg<T, MT, NS>, CU>(g, st);
        LLMQ_GROUPED_ROWS(LLMQ_GROUPED_ROWS_CASE)
#undef LLMQ_GROUPED_ROWS_CASE
    }
    return LLMQ_ERR_SHAPE;
}

}  // namespace llmq
