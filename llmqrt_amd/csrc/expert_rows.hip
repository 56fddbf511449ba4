// Rows to their experts and back.
//
//   dispatch  place[t, j] = #{ids of a smaller expert} + #{ids of the same expert before (t, j)}        offsets[e] = #{ids of an expert below e}
//             row place[t, j] of the output is token t: as it is, in int8 with a scale per token, or in e4m3 with a scale per 128 channels
//   combine   out[t] = sum_j w[t, j] y[place[t, j]] (+ shared[t])
// Ids are counted from `first`; those outside [first, first + experts) go nowhere: they have no place (-1) and are not counted.
//
// The order is that of a stable sort, so it is the same every time.  A token is read and quantized once and written top_k times.  HBM-bound: 8192 tokens of 3584
// int8 to 4 of 32 experts 38 us, of which the rows take 30 (5.8 TB/s) and their places 7.7; combined again 55 us (5.3 TB/s).  A few tokens are a launch and a chain of
// latencies: ids, places, rows (48 tokens to 4 of 64 4.0 us, combined again 2.8).
#include <algorithm>

#include "expert_tiles.h"
#include "llmq_common.h"
#include "quant_math.h"

namespace llmq {
namespace {

enum { OUT_SAME = LLMQ_NORM_SAME, OUT_I8 = LLMQ_NORM_I8_TOKEN, OUT_GROUP = LLMQ_NORM_FP8_GROUP };
constexpr int kMaxTop = 64, kMaxExperts = 4096;
constexpr int kCountAll = 4096, kIndexBits = 12;  // up to so many ids every token may count all of them for itself

struct DispatchArgs {
    const uint16_t* x;
    const int32_t* ids;
    void* rows;
    float* scale;
    int32_t *offsets, *places;
    int64_t ldx, K;
    int t0, ids_total;  // t0: token of block 0
    int tokens, top, first, experts;  // tokens: of this launch
    int wide;           // codes are stored 16 at a time
};

__device__ __forceinline__ int wave_total(int v) { return __builtin_amdgcn_readlane(wave_prefix(v), kWave - 1); }
__device__ __forceinline__ uint32_t expert_of(const int32_t* ids, int i, int first) { return (uint32_t)ids[i] - (uint32_t)first; }

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

// Many ids: a block per expert finds the places of its own.  Every wavefront has a run of the ids and goes over it twice: it counts those of smaller experts and
// of this one, and hands out places from where the runs before it end.  A run of up to U * Q * 64 ids stays in registers between the two.
// Q: ids of a lane next to each other (4: 16-byte loads); U: pieces of 64 Q ids that a run holds.  us, U = 2, 4, 8 with 16-byte loads, 8 with 4-byte ones: 8000 ids of 60
// experts 3.9 4.5 5.8 4.1, 16384 of 64 6.5 5.6 6.9 7.4, 24000 of 256 8.8 9.4 7.8 9.7.
template <int Q, int U>
__global__ __launch_bounds__(1024) void expert_places_kernel(const int32_t* __restrict__ ids, int n, int first, int experts, int32_t* __restrict__ places,
                                                             int32_t* __restrict__ offsets) {
    constexpr int NW = 1024 / kWave, PIECE = Q * kWave;  // U pieces requested before the first is used
    __shared__ int32_t s_same[NW], s_less[NW];
    const int e = blockIdx.x, lane = threadIdx.x & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int run = ((n + NW - 1) / NW + PIECE - 1) / PIECE * PIECE, lo = (int)min((int64_t)n, (int64_t)wave * run), hi = min(n - lo, run) + lo;
    uint32_t v[U][Q];
    auto load = [&](int b) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int i = b + u * PIECE + lane * Q;
            if constexpr (Q == 4) {
                const int4 w = *reinterpret_cast<const int4*>(ids + (i < n - 3 ? i : 0));  // (n > 3; the last, partial piece below)
                v[u][0] = (uint32_t)w.x, v[u][1] = (uint32_t)w.y, v[u][2] = (uint32_t)w.z, v[u][3] = (uint32_t)w.w;
            } else {
                v[u][0] = (uint32_t)ids[min(i, n - 1)];
            }
        }
        if (Q == 4 && b + U * PIECE > n - 3)  // uniform
#pragma unroll
            for (int u = 0; u < U; u++) {
                const int i = b + u * PIECE + lane * Q;
                if (i < n && i >= n - 3)
#pragma unroll
                    for (int q = 0; q < Q; q++) v[u][q] = (uint32_t)ids[min(i + q, n - 1)];
            }
    };
    // the lanes whose id q of piece u is this expert's; a piece past the run has none
    uint64_t has[U][Q];
    int less = 0, same = 0;
    auto look = [&](int b, bool count) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int at = b + u * PIECE;
#pragma unroll
            for (int q = 0; q < Q; q++) has[u][q] = 0;
            if (at >= hi) continue;  // uniform
#pragma unroll
            for (int q = 0; q < Q; q++) {
                const uint32_t id = v[u][q] - (uint32_t)first;
                const bool in = at + PIECE <= hi || at + lane * Q + q < hi;
                has[u][q] = __ballot(in && id == (uint32_t)e);
                if (count) same += (int)__popcll(has[u][q]), less += (int)__popcll(__ballot(in && id < (uint32_t)e));
            }
        }
    };
    for (int b = lo; b < hi; b += U * PIECE) load(b), look(b, true);
    if (lane == 0) s_same[wave] = same, s_less[wave] = less;
    __syncthreads();
    int before = 0, all = 0, from = 0;
#pragma unroll
    for (int w = 0; w < NW; w++) {
        before += w < wave ? s_same[w] : 0;
        all += s_same[w], from += s_less[w];
    }
    if (threadIdx.x == 0) {
        offsets[e] = from;
        if (e == experts - 1) offsets[experts] = from + all;
    }
    int at = from + before;
    for (int b = lo; b < hi; b += U * PIECE) {
        if (hi - lo > U * PIECE) load(b), look(b, false);  // (a short run is still there)
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int i = b + u * PIECE + lane * Q;
            uint64_t any = 0;
#pragma unroll
            for (int q = 0; q < Q; q++) any |= has[u][q];
            if (any) {  // uniform
                int upto = at;  // the place of the lane's first one
#pragma unroll
                for (int q = 0; q < Q; q++) upto = __builtin_amdgcn_mbcnt_hi((uint32_t)(has[u][q] >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)has[u][q], upto));
#pragma unroll
                for (int q = 0; q < Q; q++) {
                    if (has[u][q] >> lane & 1) places[i + q] = upto++;
                    at += (int)__popcll(has[u][q]);
                }
            }
            if (e == 0)
#pragma unroll
                for (int q = 0; q < Q; q++)
                    if (i + q < hi && v[u][q] - (uint32_t)first >= (uint32_t)experts) places[i + q] = -1;
        }
    }
}

// ---- very many ids: in three launches that each go over them once.  A wavefront has a run of ids; `counts` says how many of them are of each expert, then how many of
// an expert's lie in the runs before.
constexpr int kRunPieces = 4, kRunUnit = kRunPieces * kWave, kMaxRuns = 1024, kRunWaves = 2;
struct Runs {
    int n, per, runs, stride;  // ids; of a run; runs; ints of an expert in `counts`, whose last ones are the experts' totals
    int32_t* counts;
};
__device__ __forceinline__ void own_lds() {  // LDS that this wavefront alone writes and reads
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront", "local");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront", "local");
}
// the ids from b on that are in front of hi, as experts; the others are none
__device__ __forceinline__ void load_run(const int32_t* ids, int64_t b, int64_t hi, int first, uint32_t* e) {
    const int lane = threadIdx.x & (kWave - 1);
#pragma unroll
    for (int u = 0; u < kRunPieces; u++) {
        const int64_t i = b + u * kWave + lane;
        e[u] = (uint32_t)ids[i < hi ? i : hi - 1] - (uint32_t)first;
        if (i >= hi) e[u] = ~0u;
    }
}

__global__ __launch_bounds__(kRunWaves * kWave) void run_counts_kernel(const int32_t* __restrict__ ids, Runs r, int first, int experts) {
    extern __shared__ int32_t s_count[];  // of a wavefront: experts
    const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave, run = blockIdx.x * kRunWaves + wave;
    if (run >= r.runs) return;  // wavefront-uniform; no barrier follows
    int32_t* count = s_count + wave * experts;
    for (int e = lane; e < experts; e += kWave) count[e] = 0;
    own_lds();
    const int64_t lo = (int64_t)run * r.per, hi = min((int64_t)r.n, lo + r.per);
    for (int64_t b = lo; b < hi; b += kRunUnit) {
        uint32_t e[kRunPieces];
        load_run(ids, b, hi, first, e);
#pragma unroll
        for (int u = 0; u < kRunPieces; u++)
            if (e[u] < (uint32_t)experts) atomicAdd(&count[e[u]], 1);
    }
    own_lds();
    for (int e = lane; e < experts; e += kWave) r.counts[(int64_t)e * r.stride + run] = count[e];
}

// A wavefront per expert
__global__ __launch_bounds__(kWave) void run_sums_kernel(Runs r, int experts) {
    const int e = blockIdx.x, lane = threadIdx.x;
    int4* c = reinterpret_cast<int4*>(r.counts + (int64_t)e * r.stride);
    int4 v[kMaxRuns / kRunUnit];
#pragma unroll
    for (int k = 0; k < kMaxRuns / kRunUnit; k++) {
        const int i = (k * kWave + lane) * 4;
        v[k] = i < r.stride ? c[k * kWave + lane] : make_int4(0, 0, 0, 0);
        v[k].x = i < r.runs ? v[k].x : 0, v[k].y = i + 1 < r.runs ? v[k].y : 0, v[k].z = i + 2 < r.runs ? v[k].z : 0, v[k].w = i + 3 < r.runs ? v[k].w : 0;
    }
    int before = 0;
#pragma unroll
    for (int k = 0; k < kMaxRuns / kRunUnit; k++) {
        const int own = v[k].x + v[k].y + v[k].z + v[k].w, upto = before + wave_prefix(own), at = upto - own;
        if ((k * kWave + lane) * 4 < r.stride) c[k * kWave + lane] = make_int4(at, at + v[k].x, at + v[k].x + v[k].y, at + v[k].x + v[k].y + v[k].z);
        before = __builtin_amdgcn_readlane(upto, kWave - 1);
    }
    if (lane == 0) r.counts[(int64_t)experts * r.stride + e] = before;
}

// Every run hands out the places of its ids: among 64 at a time those of one expert find each other by the bits of its number, bits of them.
__global__ __launch_bounds__(kRunWaves * kWave) void run_places_kernel(const int32_t* __restrict__ ids, Runs r, int first, int experts, int bits,
                                                                       int32_t* __restrict__ places, int32_t* __restrict__ offsets) {
    extern __shared__ int32_t s_next[];  // experts' first rows; then of a wavefront: an expert's next place
    __shared__ int32_t sums[kRunWaves];
    const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave, run = blockIdx.x * kRunWaves + wave;
    for (int e = threadIdx.x; e < experts; e += kRunWaves * kWave) s_next[e] = r.counts[(int64_t)experts * r.stride + e];
    __syncthreads();
    const int total = scan_lds<kRunWaves * kWave>(s_next, experts, sums);
    if (blockIdx.x == 0) {
        for (int e = threadIdx.x; e < experts; e += kRunWaves * kWave) offsets[e] = s_next[e];
        if (threadIdx.x == 0) offsets[experts] = total;
    }
    if (run >= r.runs) return;  // wavefront-uniform; no barrier follows
    int32_t* next = s_next + (wave + 1) * experts;
    for (int e = lane; e < experts; e += kWave) next[e] = s_next[e] + r.counts[(int64_t)e * r.stride + run];
    own_lds();
    const int64_t lo = (int64_t)run * r.per, hi = min((int64_t)r.n, lo + r.per);
    for (int64_t b = lo; b < hi; b += kRunUnit) {
        uint32_t e[kRunPieces];
        uint64_t like[kRunPieces];  // the lanes with the same expert
        load_run(ids, b, hi, first, e);
#pragma unroll
        for (int u = 0; u < kRunPieces; u++) like[u] = __ballot(e[u] < (uint32_t)experts);
        for (int k = 0; k < bits; k++) {
#pragma unroll
            for (int u = 0; u < kRunPieces; u++) {
                const bool one = e[u] >> k & 1;
                const uint64_t ones = __ballot(one);
                like[u] &= one ? ones : ~ones;
            }
        }
#pragma unroll
        for (int u = 0; u < kRunPieces; u++) {
            const int64_t i = b + u * kWave + lane;
            const bool in = e[u] < (uint32_t)experts;
            int place = -1;
            if (in) place = __builtin_amdgcn_mbcnt_hi((uint32_t)(like[u] >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)like[u], next[e[u]]));
            own_lds();
            if (in && (like[u] >> lane >> 1) == 0) next[e[u]] = place + 1;  // the last of them
            own_lds();
            if (i < hi) places[i] = place;
        }
    }
}

// Whether there are so many ids that the three launches are faster than a block per expert over all of them, and how they share them.  us, a block per expert / in
// runs: 16384 ids of 64 experts 6.9 / 7.9, 32768 of 32 9.2 / 7.7, of 128 9.0 / 8.4, of 256 8.6 / 9.7, 65536 of 256 19.2 / 10.2, 262144 of 64 72 / 9.3; 16000 of 512
// 10.2 / 12.1, of 1024 17.5 / 17.6, of 4096 59 / 50.  The one grows with ids, and with experts where the chip does not hold a block of each, the other with experts.
bool in_runs(int64_t n, int64_t experts, Runs& r) {
    r.n = (int)n, r.per = (int)(((n + kMaxRuns - 1) / kMaxRuns + kRunUnit - 1) / kRunUnit * kRunUnit);
    r.runs = (int)((n + r.per - 1) / r.per), r.stride = (r.runs + 3) / 4 * 4;
    return n * std::max<int64_t>(experts, 256) > 256 * (21400 + 50 * experts);
}
size_t run_bytes(const Runs& r, int64_t experts) { return ((size_t)r.stride + 1) * experts * sizeof(int32_t); }
bool count_all(int64_t tokens, int64_t top_k) { return tokens * top_k <= kCountAll && tokens * tokens * top_k <= 1 << 22; }

// A block per token; 16 neighbouring elements per thread and piece.  ALL: every token counts all ids for itself, and one more block counts them for the
// offsets; otherwise the places are there.  NP > 0: the row stays in registers, NP pieces per thread; 0: rows of any length, read again for every copy.
template <int DT, int OUT, bool ALL, int NP, int NT>
__global__ __launch_bounds__(NT) void dispatch_kernel(DispatchArgs a) {
    constexpr int NW = NT / kWave, REGS = NP > 0 ? NP : 1, JW = 4;
    __shared__ float smem[NW];
    const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(tid / kWave);
    if constexpr (ALL) {
        if (blockIdx.x == (unsigned)a.tokens) {  // block-uniform
            __shared__ int32_t count[kMaxExperts], sums[NW];
            for (int e = tid; e < a.experts; e += NT) count[e] = 0;
            __syncthreads();
            for (int i = tid; i < a.ids_total; i += NT) {
                const uint32_t e = expert_of(a.ids, i, a.first);
                if (e < (uint32_t)a.experts) atomicAdd(&count[e], 1);
            }
            __syncthreads();
            const int total = scan_lds<NT>(count, a.experts, sums);
            for (int e = tid; e < a.experts; e += NT) a.offsets[e] = count[e];
            if (tid == 0) a.offsets[a.experts] = total;
            return;
        }
    }
    const int t = a.t0 + (int)blockIdx.x, mine = t * a.top;
    const int nchunk = (int)(a.K >> 3), npiece = (nchunk + 1) / 2;
    int goes_to = -1;  // the place of copy `lane`
    if constexpr (!ALL) goes_to = lane < a.top ? a.places[mine + lane] : -1;
    const uint4* xr = reinterpret_cast<const uint4*>(a.x + (int64_t)t * a.ldx);
    auto half = [&](int c) __attribute__((always_inline)) { return c < nchunk ? xr[c] : make_uint4(0, 0, 0, 0); };
    // the chunks of piece i: two neighbours, whose codes are 16 bytes; rows that are copied as they are: one of this half of NT chunks and one of the next
    auto chunk = [&](int i, int h) __attribute__((always_inline)) { return OUT == OUT_SAME ? i / NT * (2 * NT) + h * NT + i % NT : 2 * i + h; };
    uint4 v[REGS][2];
    if (NP > 0) {
#pragma unroll
        for (int c = 0; c < NP; c++) {
            const int i = tid + c * NT;
            v[c][0] = half(chunk(i, 0)), v[c][1] = half(chunk(i, 1));
        }
    }

    if constexpr (ALL) {
        // Expert and index in one key: a copy's place is how many keys are below its own (an id that goes nowhere is above all).  The wavefronts share JW copies
        // each and, where there are more wavefronts than that, parts of the ids.
        static_assert((int64_t)kMaxExperts << kIndexBits < 0xffffffffLL && kCountAll <= 1 << kIndexBits, "keys");
        __shared__ int32_t part[NW][kMaxTop];
        auto key = [&](int32_t id, int i) __attribute__((always_inline)) {
            return min((uint32_t)id - (uint32_t)a.first, (uint32_t)a.experts) << kIndexBits | (uint32_t)i;
        };
        const bool fours = (reinterpret_cast<uintptr_t>(a.ids) & 15u) == 0 && a.ids_total % 4 == 0;  // uniform
        const bool here = lane < a.top && key(a.ids[mine + min(lane, a.top - 1)], 0) >> kIndexBits < (uint32_t)a.experts;
        const int share = a.top <= JW ? 0 : a.top <= 2 * JW ? 1 : 31 - __builtin_clz(NW);  // 2^share wavefronts have different copies
        const int parts = NW >> share, mine_of = wave >> share;
        for (int j0 = (wave & ((1 << share) - 1)) * JW; j0 < a.top; j0 += JW << share) {
            uint32_t k0[JW];
            int n[JW];
#pragma unroll
            for (int k = 0; k < JW; k++) {
                k0[k] = j0 + k < a.top ? key(a.ids[mine + j0 + k], mine + j0 + k) : 0;
                n[k] = 0;
            }
            auto count = [&](uint32_t id) __attribute__((always_inline)) {
#pragma unroll
                for (int k = 0; k < JW; k++) n[k] += id < k0[k];
            };
            if (fours) {
#pragma unroll 4
                for (int i = (mine_of * kWave + lane) * 4; i < a.ids_total; i += parts * kWave * 4) {
                    const int4 v = *reinterpret_cast<const int4*>(a.ids + i);
                    count(key(v.x, i)), count(key(v.y, i + 1)), count(key(v.z, i + 2)), count(key(v.w, i + 3));
                }
            } else {
#pragma unroll 4
                for (int i = mine_of * kWave + lane; i < a.ids_total; i += parts * kWave) count(key(a.ids[i], i));
            }
#pragma unroll
            for (int k = 0; k < JW; k++) {
                if (j0 + k >= a.top) break;
                const int total = wave_total(n[k]);
                if (lane == 0) part[mine_of][j0 + k] = total;
            }
        }
        __syncthreads();
        if (here) {
            goes_to = 0;
#pragma unroll
            for (int w = 0; w < NW; w++) goes_to += w < parts ? part[w][lane] : 0;
        }
        if (wave == 0 && lane < a.top) a.places[mine + lane] = goes_to;
    }
    auto each_copy = [&](auto&& f) __attribute__((always_inline)) {  // f(place)
        for (int j = 0; j < a.top; j++) {
            const int p = __builtin_amdgcn_readlane(goes_to, j);
            if (p >= 0) f(p);
        }
    };
    // codes of piece i to a row
    auto store = [&](uint8_t* to, int i, uint2 q0, uint2 q1) __attribute__((always_inline)) {
        if (a.wide) {
            *reinterpret_cast<uint4*>(to + 16 * (int64_t)i) = make_uint4(q0.x, q0.y, q1.x, q1.y);
        } else {
            *reinterpret_cast<uint2*>(to + 16 * (int64_t)i) = q0;
            if (2 * i + 1 < nchunk) *reinterpret_cast<uint2*>(to + 16 * (int64_t)i + 8) = q1;
        }
    };

    // ---- the row, in its output's form, to every place
    if (OUT == OUT_SAME) {
        each_copy([&](int p) __attribute__((always_inline)) {
            uint4* to = reinterpret_cast<uint4*>((uint16_t*)a.rows + (int64_t)p * a.K);
            auto copy = [&](int i, uint4 lo, uint4 hi) __attribute__((always_inline)) {
                if (chunk(i, 0) < nchunk) to[chunk(i, 0)] = lo;
                if (chunk(i, 1) < nchunk) to[chunk(i, 1)] = hi;
            };
            if (NP > 0) {
#pragma unroll
                for (int c = 0; c < NP; c++) copy(tid + c * NT, v[c][0], v[c][1]);
            } else {
                for (int i = tid; chunk(i, 0) < nchunk; i += NT) copy(i, half(chunk(i, 0)), half(chunk(i, 1)));
            }
        });
        return;
    }
    if (OUT == OUT_I8) {  // the scale and the quotients are values of x's type, as in llmq_quant_i8_per_token
        auto most = [](uint4 lo, uint4 hi) __attribute__((always_inline)) { return max_nonneg(absmax8(lo, DT == LLMQ_BF16), absmax8(hi, DT == LLMQ_BF16)); };
        float amax = 0.f;
        if (NP > 0) {
#pragma unroll
            for (int c = 0; c < NP; c++) amax = max_nonneg(amax, most(v[c][0], v[c][1]));
        } else {
            for (int i = tid; i < npiece; i += NT) amax = max_nonneg(amax, most(half(2 * i), half(2 * i + 1)));
        }
        amax = NW > 1 ? block_max<NW>(amax, smem) : wave_max(amax);
        const float s = scale_from_amax<DT, MODE_I8>(amax), inv_s = 1.0f / s;
        const bool fin = amax < __builtin_inff() && s > 0.f;
        auto codes = [&](uint4 r) __attribute__((always_inline)) {
            return fin ? quant8<DT, MODE_I8, Q_DT, true>(r, s, inv_s) : quant8<DT, MODE_I8, Q_DT, false>(r, s, inv_s);
        };
        uint2 q[REGS][2];
        if (NP > 0) {
#pragma unroll
            for (int c = 0; c < NP; c++) q[c][0] = codes(v[c][0]), q[c][1] = codes(v[c][1]);
        }
        if (wave == 0 && goes_to >= 0) a.scale[goes_to] = s;
        each_copy([&](int p) __attribute__((always_inline)) {
            uint8_t* to = (uint8_t*)a.rows + (int64_t)p * a.K;
            if (NP > 0) {
#pragma unroll
                for (int c = 0; c < NP; c++)
                    if (tid + c * NT < npiece) store(to, tid + c * NT, q[c][0], q[c][1]);
            } else {
                for (int i = tid; i < npiece; i += NT) store(to, i, codes(half(2 * i)), codes(half(2 * i + 1)));
            }
        });
        return;
    }
    // a scale per 8 pieces, which 8 neighbouring lanes hold
    constexpr int TEAM = kTeam / 2;
    const int groups = (npiece + TEAM - 1) / TEAM;
    auto group_codes = [&](uint4 lo, uint4 hi, uint2* q) __attribute__((always_inline)) {
        float amax = max_nonneg(absmax8(lo, DT == LLMQ_BF16), absmax8(hi, DT == LLMQ_BF16));
        amax = max_nonneg(amax, lane_xor<1>(amax));
        amax = max_nonneg(amax, lane_xor<2>(amax));
        amax = max_nonneg(amax, lane_xor<4>(amax));
        const float s = scale32<MODE_F8>(amax), inv_s = 1.0f / s;
        float f[8], h[8];
        widen8<DT>(lo, f), widen8<DT>(hi, h);
        if (__all(near_ok(amax, s))) q[0] = codes8<MODE_F8, true>(f, s, inv_s), q[1] = codes8<MODE_F8, true>(h, s, inv_s);
        else q[0] = codes8<MODE_F8, false>(f, s, inv_s), q[1] = codes8<MODE_F8, false>(h, s, inv_s);
        return s;
    };
    uint2 q[REGS][2];
    float s[REGS];
    if (NP > 0) {
#pragma unroll
        for (int c = 0; c < NP; c++) s[c] = group_codes(v[c][0], v[c][1], q[c]);
    }
    each_copy([&](int p) __attribute__((always_inline)) {
        uint8_t* to = (uint8_t*)a.rows + (int64_t)p * a.K;
        float* ts = a.scale + (int64_t)p * groups;
        if (NP > 0) {
#pragma unroll
            for (int c = 0; c < NP; c++) {
                const int i = tid + c * NT;
                if (i < npiece) store(to, i, q[c][0], q[c][1]);
                if (i < npiece && i % TEAM == 0) ts[i / TEAM] = s[c];
            }
        } else {
            for (int b = 0; b < npiece; b += NT) {
                const int i = b + tid;
                s[0] = group_codes(half(2 * i), half(2 * i + 1), q[0]);
                if (i < npiece) store(to, i, q[0][0], q[0][1]);
                if (i < npiece && i % TEAM == 0) ts[i / TEAM] = s[0];
            }
        }
    });
}

// Threads for one piece each, up to 256, then pieces; us, int8 to 4 experts, threads x pieces: 8192 tokens of 896 64 x 1 18.7, 128 x 1 20.8, 256 x 1 25.4; 2000 of 2048
// 128 x 1 12.2, 256 x 1 13.1, 8192 of them 30.6 and 29.8; 8192 of 3584 256 x 1 44.1, 128 x 2 45.7, 512 x 1 44.0; 8192 of 7168 256 x 2 79, 128 x 4 81, 512 x 1 80; of 18944
// 256 x 5 187, read again for every copy by 512 285.  Longer rows, read again: by 512 463, by 256 501 (28672).  Codes stored 8 at a time: 3584 48.8, 16 at a time 44.0.
template <int DT, int OUT, bool ALL>
int launch_dispatch(const DispatchArgs& a, unsigned grid, hipStream_t st) {
    const int64_t pieces = (a.K + 15) / 16;
#define LLMQ_DISPATCH(NP, NT) hipLaunchKernelGGL((dispatch_kernel<DT, OUT, ALL, NP, NT>), dim3(grid), dim3(NT), 0, st, a)
    if (!ALL && pieces <= 64) LLMQ_DISPATCH(1, (ALL ? 256 : 64));
    else if (!ALL && pieces <= 128) LLMQ_DISPATCH(1, (ALL ? 256 : 128));
    else if (pieces <= 256) LLMQ_DISPATCH(1, 256);  // (with all ids to count, as many wavefronts as that for short rows too)
    else if (pieces <= 512) LLMQ_DISPATCH(2, 256);
    else if (pieces <= 1280) LLMQ_DISPATCH(5, 256);
    else LLMQ_DISPATCH(0, 512);
#undef LLMQ_DISPATCH
    return launch_status();
}
template <int DT>
int launch_dispatch_out(int out, bool all, const DispatchArgs& a, unsigned grid, hipStream_t st) {
    switch (out) {
        case OUT_SAME: return all ? launch_dispatch<DT, OUT_SAME, true>(a, grid, st) : launch_dispatch<DT, OUT_SAME, false>(a, grid, st);
        case OUT_I8: return all ? launch_dispatch<DT, OUT_I8, true>(a, grid, st) : launch_dispatch<DT, OUT_I8, false>(a, grid, st);
        default: return all ? launch_dispatch<DT, OUT_GROUP, true>(a, grid, st) : launch_dispatch<DT, OUT_GROUP, false>(a, grid, st);
    }
}

// ---- combine
struct CombineArgs {
    const uint16_t* y;
    const int32_t* places;
    const float* weights;
    const uint16_t* shared;
    uint16_t* out;
    int64_t ldy, lds, rows;
    uint32_t total, chunks;  // chunks of 8 channels: of the output, of a row
    int top;
};

// A thread per chunk, four rows requested before the first is used.
template <int DT>
__global__ __launch_bounds__(256) void combine_kernel(CombineArgs a) {
    const uint32_t i = blockIdx.x * 256 + threadIdx.x;
    if (i >= a.total) return;
    const int64_t t = i / a.chunks, c = (int64_t)(i - (uint32_t)t * a.chunks) * 8;
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

extern "C" size_t llmq_dispatch_experts_workspace_bytes(int64_t tokens, int64_t top_k, int64_t experts) {
    if (tokens < 1 || top_k < 1 || top_k > kMaxTop || tokens > 0x7fff0000LL / top_k || experts < 1 || experts > kMaxExperts || count_all(tokens, top_k)) return 0;
    Runs r;
    return in_runs(tokens * top_k, experts, r) ? run_bytes(r, experts) : 0;
}

extern "C" int llmq_dispatch_experts(int out, const void* x, int x_dtype, int64_t tokens, int64_t K, int64_t ldx, const int32_t* ids, int64_t top_k,
                                     int64_t first_expert, int64_t experts, void* rows, float* scale, int32_t* offsets, int32_t* places,
                                     void* workspace, size_t workspace_bytes, llmq_stream_t stream) {
    if ((out != OUT_SAME && out != OUT_I8 && out != OUT_GROUP) || (x_dtype != LLMQ_BF16 && x_dtype != LLMQ_F16)) return LLMQ_ERR_DTYPE;
    if (tokens < 0 || K < 0 || K > 0x7fffffffLL || ldx < K || (K & 7) || (ldx & 7) || top_k < 1 || top_k > kMaxTop || experts < 1 ||
        experts > kMaxExperts || first_expert < 0 || first_expert > 0x7fff0000LL || tokens > 0x7fff0000LL / top_k)
        return LLMQ_ERR_SHAPE;
    if (!offsets || (tokens > 0 && (!ids || !places || (K > 0 && (!x || !rows || (out != OUT_SAME && !scale)))))) return LLMQ_ERR_NULL;
    if (tokens > 0 && K == 0) return LLMQ_ERR_SHAPE;
    if (tokens > 0 && (!aligned16(x) || (out == OUT_SAME ? !aligned16(rows) : !aligned8(rows)))) return LLMQ_ERR_ALIGN;
    DispatchArgs a = {};
    a.x = (const uint16_t*)x, a.ids = ids, a.rows = rows, a.scale = scale, a.offsets = offsets, a.places = places;
    a.ldx = ldx, a.K = K, a.ids_total = (int)(tokens * top_k), a.top = (int)top_k, a.first = (int)first_expert, a.experts = (int)experts;
    a.wide = K % 16 == 0 && aligned16(rows);
    const hipStream_t st = (hipStream_t)stream;
    // every token counts all ids, or further launches find the places: us, counted / found (rows of 3584 int8) 512 tokens of 4 5.6 / 8.2, 1024 of 4 7.5 / 8.8, 2000 of
    // 4 14 / 8
    const bool all = count_all(tokens, top_k);
    Runs r;
    if (!all && in_runs(a.ids_total, experts, r)) {
        if (!workspace || workspace_bytes < run_bytes(r, experts)) return LLMQ_ERR_WORKSPACE;
        if (!aligned16(workspace)) return LLMQ_ERR_ALIGN;
        r.counts = (int32_t*)workspace;
        const unsigned blocks = (unsigned)((r.runs + kRunWaves - 1) / kRunWaves), threads = kRunWaves * kWave;
        int bits = 0;
        while (1 << bits < experts) bits++;
        hipLaunchKernelGGL(run_counts_kernel, dim3(blocks), dim3(threads), kRunWaves * experts * 4, st, ids, r, a.first, a.experts);
        hipLaunchKernelGGL(run_sums_kernel, dim3((unsigned)experts), dim3(kWave), 0, st, r, a.experts);
        hipLaunchKernelGGL(run_places_kernel, dim3(blocks), dim3(threads), (kRunWaves + 1) * experts * 4, st, ids, r, a.first, a.experts, bits, places, offsets);
        if (launch_status() != LLMQ_OK) return LLMQ_ERR_LAUNCH;
    } else if (!all) {
#define LLMQ_PLACES(Q, U) \
    hipLaunchKernelGGL((expert_places_kernel<Q, U>), dim3((unsigned)experts), dim3(1024), 0, st, ids, a.ids_total, a.first, a.experts, places, offsets)
        if (!aligned16(ids)) LLMQ_PLACES(1, 8);
        else if (a.ids_total <= 2 * 4 * 1024) LLMQ_PLACES(4, 2);  // (pieces of a run, ids of a lane, lanes)
        else if (a.ids_total <= 4 * 4 * 1024) LLMQ_PLACES(4, 4);
        else LLMQ_PLACES(4, 8);
#undef LLMQ_PLACES
        if (launch_status() != LLMQ_OK) return LLMQ_ERR_LAUNCH;
    }
    const int64_t step = (int64_t)1 << 21;  // tokens of a grid: 2^32 threads are too many
    int rc = LLMQ_OK;
    for (int64_t t = 0; rc == LLMQ_OK && (t < tokens || (t == 0 && all)); t += step) {
        a.t0 = (int)t, a.tokens = (int)std::min(step, tokens - t);
        const unsigned grid = (unsigned)a.tokens + (all ? 1 : 0);  // (every token counts all ids: one launch, with the block for the offsets)
        rc = x_dtype == LLMQ_BF16 ? launch_dispatch_out<LLMQ_BF16>(out, all, a, grid, st) : launch_dispatch_out<LLMQ_F16>(out, all, a, grid, st);
    }
    return rc;
}

extern "C" int llmq_combine_experts(const void* y, int dtype, int64_t rows, int64_t N, int64_t ldy, const int32_t* places, const float* weights,
                                    int64_t tokens, int64_t top_k, const void* shared, int64_t ld_shared, void* out, llmq_stream_t stream) {
    if (dtype != LLMQ_BF16 && dtype != LLMQ_F16) return LLMQ_ERR_DTYPE;
    if (rows < 0 || tokens < 0 || N < 0 || N > 0x7fffffffLL || (N & 7) || ldy < N || (ldy & 7) || top_k < 1 || top_k > kMaxTop ||
        tokens > 0x7fff0000LL / top_k || (shared && (ld_shared < N || (ld_shared & 7))))
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
        a.ldy = ldy, a.lds = ld_shared, a.rows = rows, a.chunks = (uint32_t)(N / 8), a.total = (uint32_t)(std::min(step, tokens - t) * (N / 8)), a.top = (int)top_k;
        const dim3 grid((unsigned)((a.total + 255) / 256));
        if (dtype == LLMQ_BF16) hipLaunchKernelGGL((combine_kernel<LLMQ_BF16>), grid, dim3(256), 0, (hipStream_t)stream, a);
        else hipLaunchKernelGGL((combine_kernel<LLMQ_F16>), grid, dim3(256), 0, (hipStream_t)stream, a);
        rc = launch_status();
    }
    return rc;
}
