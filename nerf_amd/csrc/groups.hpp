// Shared by the kernels that work on rows grouped by an id.
#pragma once
#include "common.hpp"

namespace nerf {
namespace grp {

constexpr int TILE_ROWS = 128;                          // rows of one tile of a group
constexpr int64_t MAX_ROWS = 0x7fffffff - TILE_ROWS;    // positions and their rounding up to a tile fit 32 bits
constexpr int64_t MAX_GROUPS = (int64_t)1 << 24;

// nerf_group_rows without its checks, for callers inside the library; keys (nullable) [n]: the sorted ids, n_groups for
// rows of no group.  workspace: workspace_bytes bytes, 256-byte aligned.
int64_t workspace_bytes(int64_t n, int64_t n_groups);
int launch_group_rows(int64_t n, const void* ids, int id_bytes, int64_t n_groups, int32_t* order, int32_t* offsets,
                      int32_t* tile_base, int32_t* keys, void* workspace, hipStream_t st);

// The group that tile `t` belongs to: the last g with tile_base[g] <= t, for 0 <= t < tile_base[n + 1], groups
// 0 .. n (n: the rows of no group).  A wave compares 64 boundaries at a time; every lane returns the same value.
// Empty groups share their boundary with the next one, and the last of them is the one that holds the tile.
__device__ __forceinline__ int group_of_tile(const int32_t* __restrict__ tile_base, int n, int t, int lane) {
    int lo = 0, count = n + 1;                          // candidates lo .. lo + count - 1; tile_base[lo] <= t holds
    while (count > 1) {
        const int step = (count + 63) >> 6;
        const int at = lane * step;
        const bool le = at < count && tile_base[lo + at] <= t;
        const int k = __popcll(__ballot(le)) - 1;       // lane 0 always holds
        lo += k * step;
        count = min(step, count - k * step);
    }
    return __builtin_amdgcn_readfirstlane(lo);
}

}  // namespace grp
}  // namespace nerf
