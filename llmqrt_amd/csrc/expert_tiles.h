// Products by experts: from a block's number to its expert, rows and channels.  Shared by the tile kernels whose rows are sorted by expert.
#pragma once
#include "llmq_common.h"

namespace llmq {
namespace {

constexpr int kExpertXcd = 8, kExpertGroupM = 8;

// sum over lanes 0 .. lane, in registers (us, by lane shuffles through LDS / so: block-scaled product of 256 rows of 64 experts 45.5 / 45.0, 700 of 90
// 8.2 / 7.5)
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

// maximum over lanes 0 .. lane of values that are not negative
template <int CTRL, int ROWS>
__device__ __forceinline__ int max_lanes(int v) { return max(v, __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xf, false)); }
__device__ __forceinline__ int wave_prefix_max(int v) {
    v = max_lanes<0x111, 0xf>(v), v = max_lanes<0x112, 0xf>(v), v = max_lanes<0x114, 0xf>(v), v = max_lanes<0x118, 0xf>(v);
    v = max_lanes<0x142, 0xa>(v);
    return max_lanes<0x143, 0xc>(v);
}

// flat block id -> place in the order of tiles: a contiguous range per XCD
__device__ __forceinline__ int place_of(int bid, int nblk) {
    const int q = nblk / kExpertXcd, r = nblk % kExpertXcd, xcd = bid % kExpertXcd, local = bid / kExpertXcd;
    return xcd < r ? xcd * (q + 1) + local : r * (q + 1) + (xcd - r) * q + local;
}
// place in one matrix's order -> (tile of rows, tile of channels): groups of kExpertGroupM tiles of rows, each of which starts its walk over the weights at
// another place, so that the XCDs do not all wait for the same weights from HBM (block-scaled product, us, all from the first channel / so: 8192 x 37888 x
// 3584 1008 / 988, on 128 x 256 tiles 1175 / 1097, 8192 x 4608 x 3584 157 / 146)
__device__ __forceinline__ void tile_of(int pid, int tiles_m, int tiles_n, int& tm, int& tn) {
    const int width = kExpertGroupM * tiles_n, group = pid / width, first = group * kExpertGroupM, size = min(tiles_m - first, kExpertGroupM);
    tm = first + (pid % width) % size;
    tn = (pid % width / size + group * tiles_n / ((tiles_m + kExpertGroupM - 1) / kExpertGroupM)) % tiles_n;
}

struct ExpertTile { int expert, row0, row_end, tn; };

// MAX: an offset counts as the largest one before it where that is larger.  -> false: that is needed and was not asked for
template <int BM, bool MAX>
__device__ __forceinline__ bool find_expert_tile(const int32_t* offsets, int experts, int M, int tiles_n, ExpertTile& tile) {
    const int lane = threadIdx.x & (kWave - 1);
    int total = 0, first, last, mine, upto, from = 0;
    uint64_t down = 0;  // an offset is below the one before
    auto count = [&](int e0, int before) __attribute__((always_inline)) {
        const bool in = e0 + lane < experts;
        first = last = 0;
        if (in) first = min(max(offsets[e0 + lane], 0), M), last = min(max(offsets[e0 + lane + 1], 0), M);  // (one load)
        if constexpr (MAX) {
            first = max(from, wave_prefix_max(first)), last = in ? max(first, last) : first;
            from = __builtin_amdgcn_readlane(last, kWave - 1);
        }
        mine = (last - first + BM - 1) / BM, upto = before + wave_prefix(mine);
    };
    for (int e0 = 0; e0 < experts; e0 += kWave) {
        count(e0, total), total = __builtin_amdgcn_readlane(upto, kWave - 1);
        if constexpr (!MAX) down |= __ballot(last < first);
    }
    if (down) return false;
    tile = ExpertTile{0, 0, 0, 0};
    const int64_t nblk = min((int64_t)gridDim.x, (int64_t)total * tiles_n);
    if (blockIdx.x >= nblk) return true;  // block-uniform
    // one expert's tiles after the other's, so that neighbours share its weights
    const int pid = place_of(blockIdx.x, (int)nblk), flat = pid / tiles_n;
    int before = 0, tiles = 1, tm;
    from = 0;
    for (int e0 = 0; e0 < experts; e0 += kWave) {
        if (experts > kWave) count(e0, before);  // (not again what is still there)
        const uint64_t has = __ballot(flat >= upto - mine && flat < upto);
        if (has) {
            const int at = __ffsll((unsigned long long)has) - 1;
            tile.expert = e0 + at;
            tile.row0 = __builtin_amdgcn_readlane(first, at), tile.row_end = __builtin_amdgcn_readlane(last, at);
            tiles = __builtin_amdgcn_readlane(mine, at), before = __builtin_amdgcn_readlane(upto, at) - tiles;
            break;
        }
        before = __builtin_amdgcn_readlane(upto, kWave - 1);
    }
    tile_of(pid - before * tiles_n, tiles, tiles_n, tm, tile.tn);
    tile.row0 += tm * BM;
    return true;
}

// A block's expert, the rows [row0, row_end) that are left of it from the block's first, and its tile of channels; false: the block has none.  Every
// wavefront counts the experts' tiles of BM rows for itself, 64 experts at a time.  Whatever the offsets hold, no row is outside [0, M) and none has two
// experts: an offset counts as the nearest in [0, M], and as the largest one before it where that is larger.  Largest ones are looked for only where an offset
// is below the one before (us, always / so: block-scaled product of 3000 rows of 300 experts, 512 x 512, 26.4 / 25.5, 4000 of 1000, 256 x 256, 50.5 / 45.5).
template <int BM>
__device__ __forceinline__ bool expert_tile(const int32_t* offsets, int experts, int M, int tiles_n, int& expert, int& row0, int& row_end, int& tn) {
    ExpertTile tile;
    if (!find_expert_tile<BM, false>(offsets, experts, M, tiles_n, tile)) find_expert_tile<BM, true>(offsets, experts, M, tiles_n, tile);
    expert = __builtin_amdgcn_readfirstlane(tile.expert);
    row0 = __builtin_amdgcn_readfirstlane(tile.row0);
    row_end = __builtin_amdgcn_readfirstlane(tile.row_end);
    tn = tile.tn;
    return row0 < row_end;  // block-uniform
}

}  // namespace
}  // namespace llmq
