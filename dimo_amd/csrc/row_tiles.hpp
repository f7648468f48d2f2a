// Tiles of rows over groups whose sizes only the device knows.
#pragma once
#include "common.hpp"

namespace dimo {

// Borders of the groups, kept inside [0, R] whatever the array holds: a bad offset gives wrong rows, never a wrong address.
__device__ __forceinline__ int clamp_offset(const int32_t *offsets, int e, int R) {
  return e == 0 ? 0 : min(max(offsets[e], 0), R);
}

struct RowTile {
  int expert;      // E: rows behind the last group; -1: no such tile
  int begin, end;  // rows of the tile
};

// An upper bound of the tiles of `rows` rows each (the rows behind the last group count as one more group).
inline int row_tile_count(int R, int E, int rows) {
  const int64_t groups = (int64_t)E + 1 < R ? (int64_t)E + 1 : R;
  return (int)(R / rows + groups);
}

// Tile number `tile` of the groups' tiles, found by every wave for itself: 64 groups at a time, their tile counts
// summed along the wave (two dependent loads and six exchanges for up to 64 groups).
__device__ __forceinline__ RowTile find_row_tile(const int32_t *__restrict__ offsets, int E, int R, int rows, int tile) {
  const int lane = threadIdx.x & 63;
  int before = 0;
  for (int e0 = 0; e0 <= E; e0 += 64) {
    const int e = e0 + lane;
    const int lo = e <= E ? clamp_offset(offsets, e, R) : R;
    const int hi = e < E ? max(lo, clamp_offset(offsets, e + 1, R)) : R;
    const int mine = (hi - lo + rows - 1) / rows;
    int scan = mine;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
      const int o = __shfl_up(scan, d);
      if (lane >= d) scan += o;
    }
    const unsigned long long past = __ballot(before + scan > tile);
    if (past) {
      const int f = __ffsll((long long)past) - 1;
      const int first = __builtin_amdgcn_readfirstlane(__shfl(before + scan - mine, f));
      const int glo = __builtin_amdgcn_readfirstlane(__shfl(lo, f)), ghi = __builtin_amdgcn_readfirstlane(__shfl(hi, f));
      RowTile t;
      t.expert = e0 + f;
      t.begin = glo + (tile - first) * rows;
      t.end = min(t.begin + rows, ghi);
      return t;
    }
    before += __builtin_amdgcn_readfirstlane(__shfl(scan, 63));
  }
  return RowTile{-1, 0, 0};
}

}  // namespace dimo
