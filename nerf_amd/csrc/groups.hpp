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

// Group tables come from the caller, who may have written into them, so nothing read from one is used as it is: positions are
// brought into [0, rows), group numbers into [0, groups], tiles into [0, max_tiles].  Tables that say something else than
// nerf_group_rows or nerf_group_offsets wrote give wrong sums, never an access outside the tensors or a loop without end.

// tiles of n rows in n_groups groups and of the rows of no group, at most
static inline int64_t max_tiles(int64_t n, int64_t n_groups) { return n / TILE_ROWS + n_groups + 1; }
__device__ __forceinline__ int checked_tiles(int tiles, int most) { return min(max(tiles, 0), most); }

// Rows of a tile that begins at position `pos` and ends at `end` or 128 rows later: at least one, all in [0, n) (n >= 1)
struct Span {
    int64_t pos;
    int count;
};
__device__ __forceinline__ Span checked_span(int64_t pos, int64_t end, int64_t n) {
    pos = pos < 0 ? 0 : pos < n ? pos : n - 1;
    const int64_t left = (end < n ? end : n) - pos;
    return {pos, left < 1 ? 1 : left < TILE_ROWS ? (int)left : TILE_ROWS};
}

// The group that tile `t` belongs to: the last g with tile_base[g] <= t, for 0 <= t < tile_base[n + 1], groups
// 0 .. n (n: the rows of no group).  A wave compares 64 boundaries at a time; every lane returns the same value.
// Empty groups share their boundary with the next one, and the last of them is the one that holds the tile.
__device__ __forceinline__ int group_of_tile(const int32_t* __restrict__ tile_base, int n, int t, int lane) {
    int lo = 0, count = n + 1;                          // candidates lo .. lo + count - 1; tile_base[lo] <= t holds
    while (count > 1) {
        const int step = (count + 63) >> 6;
        const int at = lane * step;
        const bool le = at < count && tile_base[lo + at] <= t;
        const int k = max((int)__popcll(__ballot(le)) - 1, 0);  // lane 0 always holds
        lo += k * step;
        count = min(step, count - k * step);
    }
    return __builtin_amdgcn_readfirstlane(lo);
}

}  // namespace grp
}  // namespace nerf
