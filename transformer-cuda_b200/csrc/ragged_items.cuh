// Work items of packed sequences, on the device (RaggedWork in kernels.cuh).
#pragma once

#include "kernels.cuh"

namespace b200attn {

constexpr int kRaggedTile = 128;

// First row and length of sequence i, within [0, T].
__device__ __forceinline__ int2 ragged_rows(const int* offsets, int i, int T) {
    const int a = min(max(offsets[i], 0), T), b = min(max(offsets[i + 1], a), T);
    return make_int2(a, b - a);
}

// Item x of the list in descending order of tiles, straight from the offsets of n <= kRaggedFindMax sequences; tiles = 0 where
// there are not so many. Executed by whole warps, each for itself. There are sum_i max(0, n_i - c + 1) items of c tiles or more,
// n_i being the tiles of sequence i: a bisection gives the tiles of item x, and a rank among the sequences that long its sequence.
static __device__ __noinline__ int4 ragged_find(const int* offsets, int n, int T, int x, int lane) {
    constexpr int kPer = kRaggedFindMax / 32;
    int2 rows[kPer];
    int tiles[kPer], most = 0, total = 0;
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
        const int i = k * 32 + lane;
        rows[k] = i < n ? ragged_rows(offsets, i, T) : make_int2(0, 0);
        tiles[k] = (rows[k].y + kRaggedTile - 1) / kRaggedTile;
        most = max(most, tiles[k]);
        total += tiles[k];
    }
    most = __reduce_max_sync(0xffffffffu, most);
    if (x >= __reduce_add_sync(0xffffffffu, total)) return make_int4(0, 0, 0, 0);
    auto at_least = [&](int c) {
        int sum = 0;
#pragma unroll
        for (int k = 0; k < kPer; ++k) sum += max(0, tiles[k] - c + 1);
        return __reduce_add_sync(0xffffffffu, sum);
    };
    int lo = 1, hi = most + 1;  // at_least(lo) > x >= at_least(hi)
    while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (at_least(mid) > x) lo = mid;
        else hi = mid;
    }
    int rank = x - at_least(hi);
    int4 found = make_int4(0, 0, 0, 0);
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
        const uint32_t who = __ballot_sync(0xffffffffu, tiles[k] >= lo);
        const bool mine = (who >> lane & 1u) && __popc(who & ((1u << lane) - 1u)) == rank;
        const uint32_t hit = __ballot_sync(0xffffffffu, mine);
        if (hit) {
            const int src = __ffs(hit) - 1;
            found = make_int4(__shfl_sync(0xffffffffu, rows[k].x, src), __shfl_sync(0xffffffffu, rows[k].y, src), lo, 0);
        }
        rank -= __popc(who);
    }
    return found;
}

}  // namespace b200attn
