// Block-scaled fp8 product, tile kernel.
//
//   out[m, n] = sum_b sa[m, b] sw[n / 128, b] sum_{k in block b} A[m, k] B[n, k]   (+ bias[n])        A, B e4m3, blocks of 128 of K
//
// Each block of K is one v_mfma_f32_16x16x128_f8f6f4 per 16 x 16 outputs that starts from zero; its four results per lane are scaled into the
// fp32 accumulators on the vector unit.  The weights feed the MFMA's row operand, so a lane holds one token (lane % 16) and four
// channels, and its factor sa sw is one register for all channel tiles of the token.
#include <type_traits>

#include "gemm_block.h"

namespace llmq {
namespace {

typedef int v8i __attribute__((ext_vector_type(8)));
typedef float v4f __attribute__((ext_vector_type(4)));

constexpr int kNumXcd = 8, kGroupM = 8;

template <int B, int E, class F>
__device__ __forceinline__ void unrolled(F&& f) {
    if constexpr (B < E) {
        f(std::integral_constant<int, B>{});
        unrolled<B + 1, E>(f);
    }
}

// A block owns BM tokens x BN channels.  KS groups of WM x WN wavefronts share its blocks of K among them, one each per stage; a wavefront owns
// (16 TM) x (16 TN) outputs, and the groups' sums are added at the end.
template <int BM_, int BN_, int WM_, int WN_, int NS_, int KS_>
struct TileCfg {
    static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_;
    static constexpr int KS = KS_, NG = WM * WN * kWave, NT = NG * KS;  // threads of a group, of the block
    static constexpr int WTM = BM / WM, WTN = BN / WN, TM = WTM / 16, TN = WTN / 16, TT = TM * TN;
    static constexpr int A_LOADS = BM * 8 / NG, B_LOADS = BN * 8 / NG, LPT = A_LOADS + B_LOADS + 1;  // per thread and stage, one of scales
    static constexpr int DATA = (BM + BN) * 128, SUB = DATA + NG * 4, STAGE = KS * SUB;  // bytes; a group's part: its operands, a slot for a scale per thread
    static constexpr int NS = NS_;  // LDS stages
    static constexpr int LDS_BYTES = NS * STAGE;
    static_assert(TM % 2 == 0 && TN >= 2 && TT % 4 == 0, "fragment parity, pending products");
    static_assert(BM + (BN + 127) / 128 <= NG && 128 % WTN == 0 && (NG / 8) % 16 == 0, "scale slots, a wavefront's channels in one block, swizzle");
    static_assert(A_LOADS * NG == BM * 8 && B_LOADS * NG == BN * 8 && (NS - 2) * LPT < 64, "even pieces, vmcnt");
    static_assert(LDS_BYTES <= 160 * 1024 && (KS - 1) * BM * BN * 4 <= LDS_BYTES, "stages, the groups' sums");
};

// LDS place of 16-byte chunk c of row r: 16 rows of one chunk fall on 16 places
__device__ __forceinline__ int chunk_at(int r, int c) { return (r * 8 + (c ^ ((r >> 1) & 7))) * 16; }

// the first `left` of eight 16-bit outputs, to any even address
__device__ __forceinline__ void store8(uint16_t* to, uint4 v, int left) {
    typedef uint32_t u4v __attribute__((ext_vector_type(4)));
    typedef u4v u4any __attribute__((aligned(2)));
    if (left >= 8) {
        __builtin_nontemporal_store(u4v{v.x, v.y, v.z, v.w}, reinterpret_cast<u4any*>(to));
    } else {
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int e = 0; e < 7; e++)
            if (e < left) to[e] = (uint16_t)(w[e / 2] >> (16 * (e & 1)));
    }
}

// sum over lanes 0 .. lane, in registers (us, by lane shuffles through LDS / so: 256 rows of 64 experts 45.5 / 45.0, 700 of 90 8.2 / 7.5)
template <int CTRL, int ROWS>
__device__ __forceinline__ int plus_lanes(int v) {  // of the rows of 16 lanes in ROWS; where there is none, plus zero
    return v + __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xf, false);
}
__device__ __forceinline__ int wave_prefix(int v) {
    v = plus_lanes<0x111, 0xf>(v);  // the lane before, in a row of 16
    v = plus_lanes<0x112, 0xf>(v);
    v = plus_lanes<0x114, 0xf>(v);
    v = plus_lanes<0x118, 0xf>(v);
    v = plus_lanes<0x142, 0xa>(v);  // rows 1 and 3: the last lane of the row before
    return plus_lanes<0x143, 0xc>(v);  // rows 2 and 3: lane 31
}

// flat block id -> place in the order of tiles: a contiguous range per XCD
__device__ __forceinline__ int place_of(int bid, int nblk) {
    const int q = nblk / kNumXcd, r = nblk % kNumXcd, xcd = bid % kNumXcd, local = bid / kNumXcd;
    return xcd < r ? xcd * (q + 1) + local : r * (q + 1) + (xcd - r) * q + local;
}
// place in one matrix's order -> (tile of rows, tile of channels): groups of kGroupM tiles of rows, each of which starts its walk over the weights at
// another place, so that the XCDs do not all wait for the same weights from HBM (us, all from the first channel / so: 8192 x 37888 x 3584 1008 / 988,
// on 128 x 256 tiles 1175 / 1097, 8192 x 4608 x 3584 157 / 146)
__device__ __forceinline__ void tile_of(int pid, int tiles_m, int tiles_n, int& tm, int& tn) {
    const int width = kGroupM * tiles_n, group = pid / width, first = group * kGroupM, size = min(tiles_m - first, kGroupM);
    tm = first + (pid % width) % size;
    tn = (pid % width / size + group * tiles_n / ((tiles_m + kGroupM - 1) / kGroupM)) % tiles_n;
}

// TAIL: K, or a split's share of it, is not made of whole blocks for every group
template <class C, bool GROUPED, bool SPLIT, bool TAIL>
__global__ __launch_bounds__(C::NT) void block_tile_kernel(BlockArgs g) {
    extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
    constexpr int TM = C::TM, TN = C::TN, NG = C::NG, NS = C::NS, TT = C::TT, KS = C::KS;
    const int group = KS > 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x / NG) : 0, tid = threadIdx.x - group * NG;
    const int lane = tid & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(tid / kWave);  // of the group
    const int wm = wave / C::WN, wn = wave % C::WN, l16 = lane & 15, kq = lane >> 4;
    const int tiles_n = (g.N + C::BN - 1) / C::BN;

    // ---- the block's rows [row0, row_end) and channels from n0
    int tm, tn, row0, row_end, expert = 0;
    if (!GROUPED) {
        const int tiles_m = (g.M + C::BM - 1) / C::BM;
        tile_of(place_of(blockIdx.x, gridDim.x), tiles_m, tiles_n, tm, tn);
        row0 = tm * C::BM, row_end = g.M;
    } else {
        // the experts' tiles of rows, counted by every wavefront for itself: 64 experts at a time
        int total = 0, first, last, mine, upto;
        auto count = [&](int e0, int before) __attribute__((always_inline)) {
            first = last = 0;
            if (e0 + lane < g.experts) expert_rows(g, e0 + lane, first, last);
            mine = (last - first + C::BM - 1) / C::BM, upto = before + wave_prefix(mine);
        };
        for (int e0 = 0; e0 < g.experts; e0 += kWave) count(e0, total), total = __builtin_amdgcn_readlane(upto, kWave - 1);
        const int64_t nblk = min((int64_t)gridDim.x, (int64_t)total * tiles_n);
        if (blockIdx.x >= nblk) return;  // block-uniform
        // one expert's tiles after the other's, so that neighbours share its weights
        const int pid = place_of(blockIdx.x, (int)nblk), flat = pid / tiles_n;
        int before = 0, tiles = 1;
        row0 = row_end = 0;
        for (int e0 = 0; e0 < g.experts; e0 += kWave) {
            if (g.experts > kWave) count(e0, before);  // (not again what is still there)
            const uint64_t has = __ballot(flat >= upto - mine && flat < upto);
            if (has) {
                const int at = __ffsll((unsigned long long)has) - 1;
                expert = e0 + at;
                row0 = __builtin_amdgcn_readlane(first, at), row_end = __builtin_amdgcn_readlane(last, at);
                tiles = __builtin_amdgcn_readlane(mine, at), before = __builtin_amdgcn_readlane(upto, at) - tiles;
                break;
            }
            before = __builtin_amdgcn_readlane(upto, kWave - 1);
        }
        tile_of(pid - before * tiles_n, tiles, tiles_n, tm, tn);
        row0 += tm * C::BM;
        expert = __builtin_amdgcn_readfirstlane(expert);
        row0 = __builtin_amdgcn_readfirstlane(row0);
        row_end = __builtin_amdgcn_readfirstlane(row_end);
        if (row0 >= row_end) return;  // block-uniform
    }
    const int n0 = tn * C::BN;
    const int kb0 = SPLIT ? blockIdx.y * g.blocks_per_split : 0, kb1 = SPLIT ? min(g.KB, kb0 + g.blocks_per_split) : g.KB;
    const int kfull = (min(kb1, g.K / kScaleBlock) - kb0) / KS;  // whole blocks of each group
    const uint8_t* B = g.B + (int64_t)expert * g.N * g.ldb;
    const float* sw = g.sw + (int64_t)expert * g.NB * g.KB;

    // ---- global -> LDS.  A thread's pieces are row tid / 8 + i NG / 8 of the tile, LDS slot tid % 8, which holds the row's chunk
    // slot ^ swizzle.  Rows past the end are the last row again.
    const int ld_row = tid / 8, ld_chunk = (tid % 8) ^ ((ld_row >> 1) & 7);
    uint32_t off[C::A_LOADS + C::B_LOADS];
#pragma unroll
    for (int i = 0; i < C::A_LOADS; i++) off[i] = (uint32_t)min(ld_row + i * (NG / 8), row_end - 1 - row0) * (uint32_t)g.lda + ld_chunk * 16;
#pragma unroll
    for (int i = 0; i < C::B_LOADS; i++) off[C::A_LOADS + i] = (uint32_t)min(ld_row + i * (NG / 8), g.N - 1 - n0) * (uint32_t)g.ldb + ld_chunk * 16;
    const uint8_t* a_base = g.A + (int64_t)row0 * g.lda;
    const uint8_t* b_base = B + (int64_t)n0 * g.ldb;
    // scale slot tid: tokens in the order in which a lane reads them (its TM tokens together), then the blocks of channels
    const float* s_ptr;
    if (tid < C::BM) {
        const int w = tid / C::WTM, r = tid % C::WTM, token = w * C::WTM + (r % TM) * 16 + r / TM;
        s_ptr = g.sa + (int64_t)min(row0 + token, row_end - 1) * g.KB;
    } else {
        s_ptr = sw + (int64_t)min(n0 / kScaleBlock + min(tid - C::BM, (C::BN - 1) / kScaleBlock), g.NB - 1) * g.KB;
    }
    const uint8_t* sub = smem + group * C::SUB;  // the group's part of stage 0
    const uint32_t lds_base = (uint32_t)(uintptr_t)((__attribute__((address_space(3))) void*)smem) + (uint32_t)group * C::SUB;
    // The walk over K starts at an eighth that follows from the tile of channels and wraps around: the XCDs work on different channels, and so do not
    // all ask for the same part of the rows at once, which lie the same distance apart and fall on few memory channels (us, from 0 / so: 777 x 3584 x
    // 18944 on 128 x 256 tiles 130 / 115, in two splits 82 / 76).  A channel's sums have one order for every token of a call.
    int ld_kb = kb0 + group + tn * kNumXcd / tiles_n * kfull / kNumXcd * KS;
    // What the groups' whole blocks leave of this split comes last: at most a block for each group, one of them ragged.  Its missing chunks are read as
    // the block's first one (a group without a block: of any), and zeros take their place in the weights' operand; what the tokens have there belongs to the
    // same row, so where it is NaN the result is too.  A group without a block multiplies nothing: the scales that it read may be infinite.
    // It has a place of its own behind the loop below, so that the others' loads have no part in it (us, each load's offset corrected in the loop / so: 8192 x
    // 37888 x 3584 1055 / 990, 1000 x 4608 x 3584 26.2 / 25.4).
    const bool rest = TAIL && kb0 + kfull * KS < kb1;  // block-uniform
    const int kall = kfull + (rest ? 1 : 0), tail_kb = min(kb0 + kfull * KS + group, g.KB - 1);
    const int left = kb0 + kfull * KS + group < kb1 ? min(g.K - (kb0 + kfull * KS + group) * kScaleBlock, kScaleBlock) : 0;
    auto next_kb = [&]() __attribute__((always_inline)) {
        ld_kb += KS;
        if (ld_kb >= kb0 + kfull * KS) ld_kb -= kfull * KS;
    };
    auto last_kb = [&]() __attribute__((always_inline)) {  // the last block of all is requested next
        if (!TAIL) return;
        ld_kb = rest ? tail_kb : ld_kb;
        const uint32_t back = rest && ld_chunk * 16 >= min(left, g.K - tail_kb * kScaleBlock) ? ld_chunk * 16 : 0;
#pragma unroll
        for (int i = 0; i < C::A_LOADS + C::B_LOADS; i++) off[i] -= back;
    };
    auto issue = [&](int stage, auto d_c) __attribute__((always_inline)) {  // piece d of block ld_kb
        constexpr int d = decltype(d_c)::value;
        const uint32_t to = lds_base + (uint32_t)stage * C::STAGE;
        if constexpr (d < C::A_LOADS + C::B_LOADS) {
            const uint8_t* base = (d < C::A_LOADS ? a_base : b_base) + (int64_t)ld_kb * kScaleBlock;
            const uint32_t m0v = to + (uint32_t)d * (NG * 16) + (uint32_t)wave * 1024;
            asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(m0v), "v"(off[d]), "s"(base) : "memory", "m0");
        } else {
            const float* p = s_ptr + ld_kb;
            const uint32_t m0v = to + C::DATA + (uint32_t)wave * 256;
            asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off" ::"s"(m0v), "v"(p) : "memory", "m0");
        }
    };
    auto lds_barrier = []() __attribute__((always_inline)) {  // orders LDS traffic only: loads stay in flight across it
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
    };

    // ---- LDS -> operands
    const int a_row = wm * C::WTM + l16, b_row = C::BM + wn * C::WTN + l16;
    auto fragment = [&](const uint8_t* st, int row) __attribute__((always_inline)) {
        const uint4 lo = *reinterpret_cast<const uint4*>(st + chunk_at(row, kq)), hi = *reinterpret_cast<const uint4*>(st + chunk_at(row, kq + 4));
        return v8i{(int)lo.x, (int)lo.y, (int)lo.z, (int)lo.w, (int)hi.x, (int)hi.y, (int)hi.z, (int)hi.w};
    };
    v8i a[2], b[TN];
    v4f acc[TM][TN], p[4];
    float s[TM], s_next[TM], w_next;
    auto read_scales = [&](const uint8_t* st) __attribute__((always_inline)) {
        const float* f = reinterpret_cast<const float*>(st + C::DATA);
#pragma unroll
        for (int i = 0; i < TM; i++) s_next[i] = f[wm * C::WTM + l16 * TM + i];
        w_next = f[C::BM + wn * C::WTN / kScaleBlock];
    };
#pragma unroll
    for (int i = 0; i < TM; i++)
#pragma unroll
        for (int j = 0; j < TN; j++) acc[i][j] = v4f{0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < 4; i++) p[i] = v4f{0, 0, 0, 0};
    auto scale_in = [&](auto t_c, float f) __attribute__((always_inline)) {
        constexpr int t = decltype(t_c)::value, i = t / TN, j = t % TN;
#pragma unroll
        for (int e = 0; e < 4; e++) acc[i][j][e] = fmaf(p[t & 3][e], f, acc[i][j][e]);
    };
    auto wait_loads = [](int younger) __attribute__((always_inline)) {  // until at most `younger` later stages are in flight
        if (NS > 3 && younger >= 2) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(NS > 3 ? 2 * C::LPT : 0) : "memory");
        else if (NS > 2 && younger == 1) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(NS > 2 ? C::LPT : 0) : "memory");
        else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    };

    // One block of K, kt.  A product's results are scaled in DELAY MFMAs later, so that the matrix cores never wait for the vector unit; the operands of
    // the next row of tiles are read under the MFMAs of this one, and those of the next block under the last row, behind the barrier that
    // publishes its stage and frees this one.  The priority alternates every two MFMAs, so that the two wavefronts of a SIMD take turns at its
    // matrix core and vector unit.  REST: the pieces of block kt + NS - 1 that the last call did not request (FIRST: this one requests
    // the others of kt + NS, into the stage that it frees).
    // (us, 2 MFMAs later without priorities / 3 with: 8192 x 37888 x 3584 951 / 930, 4096 x 3584 x 18944 228 / 222, 777 x 3584 x 18944 on 128 x 256 tiles 104 / 97)
    constexpr int DELAY = TT > 4 ? 3 : 2;  // (four tiles: s_next is the next block's from the third on)
    constexpr int PER = (C::LPT + TT - 1) / TT, EARLY = TN * PER < C::LPT ? TN * PER : C::LPT;
    static_assert(EARLY + (TT - TN) * PER >= C::LPT, "all of a block is requested before the wait that counts it");
    auto k_block = [&](const uint8_t* st, const uint8_t* next, int stage, int prev, int younger, auto rest_c, auto first_c, auto next_c, auto last_c) __attribute__((always_inline)) {
        constexpr bool REST = decltype(rest_c)::value, FIRST = decltype(first_c)::value, NEXT = decltype(next_c)::value, LAST = decltype(last_c)::value;
        unrolled<0, TT>([&](auto t_c) __attribute__((always_inline)) {
            constexpr int t = decltype(t_c)::value, i = t / TN, j = t % TN;
            if constexpr (NEXT && i == TM - 1 && j == 0) {
                if constexpr (REST) next_kb();
                if constexpr (LAST) last_kb();
                wait_loads(younger);
                lds_barrier();
            }
            if constexpr (t % 2 == 0) __builtin_amdgcn_s_setprio(t % 4 == 0);
            p[t & 3] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(b[j], a[i & 1], v4f{0, 0, 0, 0}, 0, 0, 0, 0, 0, 0);
            if constexpr (t == DELAY) {  // until here s is the last block's; from the last row on s_next is the next one's
#pragma unroll
                for (int k = 0; k < TM; k++) s[k] = s_next[k] * w_next;
            }
            if constexpr (j == 0 && i + 1 < TM) a[(i + 1) & 1] = fragment(st, a_row + (i + 1) * 16);
            if constexpr (NEXT && i == TM - 1) {
                if constexpr (j == 0) a[0] = fragment(next, a_row);
                b[j] = fragment(next, b_row + j * 16);
                if constexpr (j == 0) read_scales(next);
            }
            if constexpr (t >= DELAY) scale_in(std::integral_constant<int, t - DELAY>{}, s[(t - DELAY) / TN]);
            else scale_in(std::integral_constant<int, TT - DELAY + t>{}, s[(TT - DELAY + t) / TN]);
            constexpr int D = i == TM - 1 ? j * PER : EARLY + t * PER;
            if constexpr (i == TM - 1 ? FIRST : REST)
                unrolled<(D < C::LPT ? D : C::LPT), (D + PER < C::LPT ? D + PER : C::LPT)>(
                    [&](auto d) __attribute__((always_inline)) { issue(i == TM - 1 ? stage : prev, d); });
            __builtin_amdgcn_sched_barrier(0);
        });
    };
    auto first_operands = [&](const uint8_t* st) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < TN; j++) b[j] = fragment(st, b_row + j * 16);
        a[0] = fragment(st, a_row);
        read_scales(st);
    };
#pragma unroll
    for (int i = 0; i < TM; i++) s[i] = 0.f;

    const std::true_type yes;
    const std::false_type no;
    // all of the K loop; step(stage, next, prev, younger, REST, FIRST, NEXT, LAST) does a block
    auto drive = [&](auto&& ready, auto&& step) __attribute__((always_inline)) {
        unrolled<0, NS - 1>([&](auto n_c) __attribute__((always_inline)) {
            constexpr int n = decltype(n_c)::value;
            if (n < kall) {
                if (n == kall - 1) last_kb();
                unrolled<0, C::LPT>([&](auto d) __attribute__((always_inline)) { issue(n, d); });
                next_kb();
            }
        });
        if (kall > 0) {
            wait_loads(min(kall, NS - 1) - 1);
            lds_barrier();
            ready();
        }
        if (NS - 1 < kall) {
            if (NS == kall) last_kb();
            unrolled<0, EARLY>([&](auto d) __attribute__((always_inline)) { issue(NS - 1, d); });
        }
        int stage = 0, kt = 0;
        auto one = [&](auto rest_c, auto first_c, auto next_c, auto last_c, int younger) __attribute__((always_inline)) {
            const int next = stage == NS - 1 ? 0 : stage + 1, prev = stage == 0 ? NS - 1 : stage - 1;
            step(stage, next, prev, younger, rest_c, first_c, next_c, last_c);
            stage = next, kt++;
        };
#pragma unroll 1
        while (kt + NS + (TAIL ? 1 : 0) < kall) one(yes, yes, yes, no, NS - 2);
        if constexpr (TAIL) {
            if (kt + NS < kall) one(yes, yes, yes, yes, NS - 2);
        }
        if (kt + NS == kall) one(yes, no, yes, no, NS - 2);
#pragma unroll 1
        while (kt + 1 < kall) one(no, no, yes, no, kall - 2 - kt);
        if (kt < kall) one(no, no, no, no, 0);
    };
    if (row0 + wm * C::WTM >= row_end || n0 + wn * C::WTN >= g.N) {
        // a wavefront whose rows or channels all lie behind the last one loads its pieces and waits with the others, and multiplies nothing
        // (32768 rows on 28 of 32 experts, 4864 x 3584, 256-row tiles: 672 us multiplying, 606 not)
        drive([] {}, [&](int stage, int, int prev, int younger, auto rest_c, auto first_c, auto next_c, auto last_c) __attribute__((always_inline)) {
            if constexpr (decltype(rest_c)::value) {
                unrolled<EARLY, C::LPT>([&](auto d) __attribute__((always_inline)) { issue(prev, d); });
                next_kb();
                if constexpr (decltype(last_c)::value) last_kb();
            }
            if constexpr (decltype(next_c)::value) {
                wait_loads(younger);
                lds_barrier();
            }
            if constexpr (decltype(first_c)::value) unrolled<0, EARLY>([&](auto d) __attribute__((always_inline)) { issue(stage, d); });
        });
        if constexpr (KS > 1) lds_barrier(), lds_barrier(), lds_barrier();
        else if (!SPLIT) lds_barrier();
        return;
    }
    drive([&]() __attribute__((always_inline)) { first_operands(sub); },
          [&](int stage, int next, int prev, int younger, auto rest_c, auto first_c, auto next_c, auto last_c) __attribute__((always_inline)) {
              if (TAIL && !decltype(next_c)::value && rest) {  // the last block: a lane's chunks kq and kq + 4 of it
                  if (KS > 1 && left == 0) return;  // (one group always has a block here); the products before are scaled in behind the loop
                  const int lo = kq * 16 < left ? -1 : 0, hi = (kq + 4) * 16 < left ? -1 : 0;
#pragma unroll
                  for (int j = 0; j < TN; j++)
#pragma unroll
                      for (int e = 0; e < 8; e++) b[j][e] &= e < 4 ? lo : hi;
              }
              k_block(sub + stage * C::STAGE, sub + next * C::STAGE, stage, prev, younger, rest_c, first_c, next_c, last_c);
          });
    unrolled<TT - DELAY, TT>([&](auto t_c) __attribute__((always_inline)) { scale_in(t_c, s[decltype(t_c)::value / TN]); });
    if constexpr (KS > 1) {  // the groups' sums, in order
        v4f* sums = reinterpret_cast<v4f*>(smem) + ((group - 1) * (NG / kWave) + wave) * TT * kWave + lane;
        lds_barrier();  // every wavefront has read its last operands
        if (group > 0)
#pragma unroll
            for (int t = 0; t < TT; t++) sums[t * kWave] = acc[t / TN][t % TN];
        lds_barrier();
        if (group == 0)
#pragma unroll
            for (int k = 1; k < KS; k++)
#pragma unroll
                for (int t = 0; t < TT; t++) acc[t / TN][t % TN] += sums[(k * (NG / kWave) * TT + t) * kWave];
        lds_barrier();  // and their sums: the outputs take their place
        if (group > 0) return;
    }

    // ---- a lane holds token l16 of each tile of tokens and channels 4 kq .. + 3 of each tile of channels
    const int wm0 = row0 + wm * C::WTM, wn0 = n0 + wn * C::WTN;
    if constexpr (SPLIT) {
        const int64_t ldp = partial_ld(g.N);  // whole 32-byte pieces: a piece that starts in the row ends in its padding
        float* part = g.partials + (int64_t)blockIdx.y * g.M * ldp;
#pragma unroll
        for (int i = 0; i < TM; i++) {
            const int m = wm0 + i * 16 + l16;
            if (m >= row_end) continue;
#pragma unroll
            for (int j = 0; j < TN; j++) {
                const int n = wn0 + j * 16 + kq * 4;
                if (n < g.N) *reinterpret_cast<v4f*>(part + (int64_t)m * ldp + n) = acc[i][j];
            }
        }
    } else {
        const bool bf16 = g.out_dtype == LLMQ_BF16;
        float bb[TN][4];
#pragma unroll
        for (int j = 0; j < TN; j++)
#pragma unroll
            for (int e = 0; e < 4; e++)
                bb[j][e] = g.bias ? load_as_f32(g.bias, g.bias_dtype, (int64_t)expert * g.N + min(wn0 + j * 16 + kq * 4 + e, g.N - 1)) : 0.f;
        // Through LDS, so that a store covers whole lines of a row: a wavefront's outputs go to a region of its own, 16-byte chunk c of row r at
        // chunk c ^ (r % CH), and come back 16 bytes per lane, CH lanes a row.  (8 bytes per lane from the registers: 8192 x 37888 x 3584 1403 us,
        // so 1130.)  Rows of an odd number of channels start at any even address; the stores are as wide there (2 bytes at a time from the
        // registers: 4138 x 2847 x 944 40.6 us, so 25.8).
        constexpr int CH = C::WTN / 8, RPI = kWave / CH;
        static_assert(C::WTM * C::WTN * 2 * (NG / kWave) <= C::LDS_BYTES, "outputs fit in the ring");
        if constexpr (KS == 1) lds_barrier();  // every wavefront has read its last operands
        uint8_t* mine = smem + wave * (C::WTM * C::WTN * 2);
#pragma unroll
        for (int i = 0; i < TM; i++)
#pragma unroll
            for (int j = 0; j < TN; j++) {
                const int r = i * 16 + l16;
                float v[4];
#pragma unroll
                for (int e = 0; e < 4; e++) v[e] = acc[i][j][e] + bb[j][e];
                *reinterpret_cast<uint2*>(mine + (r * CH + ((2 * j + (kq >> 1)) ^ (r % CH))) * 16 + (kq & 1) * 8) =
                    bf16 ? make_uint2(Lo<LLMQ_BF16>::pack2(v[0], v[1]), Lo<LLMQ_BF16>::pack2(v[2], v[3]))
                         : make_uint2(Lo<LLMQ_F16>::pack2(v[0], v[1]), Lo<LLMQ_F16>::pack2(v[2], v[3]));
            }
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront", "local");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront", "local");
        const int c = lane % CH, n = wn0 + c * 8;
#pragma unroll
        for (int k = 0; k < C::WTM / RPI; k++) {
            const int r = k * RPI + lane / CH;
            const uint4 v = *reinterpret_cast<const uint4*>(mine + (r * CH + (c ^ (r % CH))) * 16);
            if (wm0 + r < row_end) store8(reinterpret_cast<uint16_t*>(g.out) + (int64_t)(wm0 + r) * g.ldo + n, v, g.N - n);
        }
    }
}

// The splits' sums in order, bias, rounding; 8 channels per thread, all splits requested before the first is used.  (us with two splits of 777 x 3584: 4
// channels per thread 7.9, so 6.2; partial sums stored past the L2: products 2-10 % slower.)
__global__ __launch_bounds__(256) void block_reduce_kernel(BlockArgs g, int splits) {
    const int64_t ldp = partial_ld(g.N), per_row = ldp / 8, i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= per_row * g.M) return;
    const int m = (int)((uint64_t)i <= 0xffffffffu ? (uint32_t)i / (uint32_t)per_row : i / per_row), n = (int)(i - (int64_t)m * per_row) * 8;
    const int64_t plane = (int64_t)g.M * ldp;
    const float* p = g.partials + (int64_t)m * ldp + n;
    float v[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    v4f q[kMostSplits][2];  // (past the last channel: padding that nobody wrote, and nobody keeps)
#pragma unroll
    for (int k = 0; k < kMostSplits; k++)
        if (k < splits) {  // uniform
            q[k][0] = *reinterpret_cast<const v4f*>(p + k * plane);
            q[k][1] = *(reinterpret_cast<const v4f*>(p + k * plane) + 1);
        }
#pragma unroll
    for (int k = 0; k < kMostSplits; k++)
        if (k < splits)
#pragma unroll
            for (int e = 0; e < 8; e++) v[e] += q[k][e / 4][e % 4];
    if (g.bias)
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] += load_as_f32(g.bias, g.bias_dtype, min(n + e, g.N - 1));
    const bool bf16 = g.out_dtype == LLMQ_BF16;
    uint32_t w[4];
#pragma unroll
    for (int e = 0; e < 4; e++) w[e] = bf16 ? Lo<LLMQ_BF16>::pack2(v[2 * e], v[2 * e + 1]) : Lo<LLMQ_F16>::pack2(v[2 * e], v[2 * e + 1]);
    store8(reinterpret_cast<uint16_t*>(g.out) + (int64_t)m * g.ldo + n, make_uint4(w[0], w[1], w[2], w[3]), g.N - n);
}

template <class C, bool GROUPED, bool SPLIT, bool TAIL>
int launch_tile(const BlockArgs& g, int splits, hipStream_t st) {
    auto kernel = block_tile_kernel<C, GROUPED, SPLIT, TAIL>;
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
    const int64_t tiles_n = (g.N + C::BN - 1) / C::BN;
    // by experts: each may end with a tile that is not full
    const int64_t tiles_m = GROUPED ? g.M / C::BM + (g.experts < g.M ? g.experts : g.M) : (g.M + C::BM - 1) / C::BM;
    if (tiles_m * tiles_n * C::NT > 0xffffffffLL) return LLMQ_ERR_SHAPE;  // threads of a grid
    hipLaunchKernelGGL(kernel, dim3((unsigned)(tiles_m * tiles_n), SPLIT ? splits : 1), dim3(C::NT), C::LDS_BYTES, st, g);
    if (launch_status() != LLMQ_OK) return LLMQ_ERR_LAUNCH;
    if (SPLIT) {
        const int64_t n = partial_ld(g.N) / 8 * g.M;
        if (n > 0xffffff00LL || splits > kMostSplits) return LLMQ_ERR_SHAPE;
        hipLaunchKernelGGL(block_reduce_kernel, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, st, g, splits);
        return launch_status();
    }
    return LLMQ_OK;
}

template <class C, bool TAIL>
int launch_kind(const BlockArgs& g, int splits, hipStream_t st) {
    if (g.offsets) return launch_tile<C, true, false, TAIL>(g, 1, st);
    return splits > 1 ? launch_tile<C, false, true, TAIL>(g, splits, st) : launch_tile<C, false, false, TAIL>(g, 1, st);
}

template <class C>
int launch_cfg(const BlockArgs& g, int splits, hipStream_t st) {
    const bool whole = g.K % kScaleBlock == 0 && g.KB % C::KS == 0 && (splits == 1 || g.blocks_per_split % C::KS == 0);
    return whole ? launch_kind<C, false>(g, splits, st) : launch_kind<C, true>(g, splits, st);
}

}  // namespace

int launch_block_tile(int cfg, int splits, const BlockArgs& g, hipStream_t st) {
    switch (cfg) {
        case 0: return launch_cfg<TileCfg<256, 256, 2, 4, 2, 1>>(g, splits, st);
        case 1: return launch_cfg<TileCfg<128, 256, 2, 4, 3, 1>>(g, splits, st);
        case 2: return launch_cfg<TileCfg<64, 256, 2, 4, 3, 1>>(g, splits, st);
        case 3: return launch_cfg<TileCfg<64, 128, 2, 2, 3, 1>>(g, splits, st);
        case 4: return launch_cfg<TileCfg<32, 128, 1, 4, 3, 1>>(g, splits, st);
        case 5: return launch_cfg<TileCfg<64, 64, 2, 2, 4, 1>>(g, splits, st);
        case 6: return launch_cfg<TileCfg<64, 128, 2, 2, 3, 2>>(g, splits, st);
        case 7: return launch_cfg<TileCfg<64, 64, 2, 2, 4, 2>>(g, splits, st);
    }
    return LLMQ_ERR_SHAPE;
}

}  // namespace llmq
