// Tiles of rows over groups whose sizes only the device knows.
#pragma once
#include "common.hpp"

namespace dimo {

// Borders of the groups, kept inside [0, R] whatever the array holds: a bad offset gives wrong rows, never a wrong address.
// No offsets: one group of all rows.
__device__ __forceinline__ int clamp_offset(const int32_t *offsets, int e, int R) {
  return e == 0 ? 0 : offsets ? min(max(offsets[e], 0), R) : R;
}

struct RowTile {
  int expert;      // E: rows behind the last group; -1: no such tile
  int begin, end;  // rows of the tile
  int number;      // the tile's number among all groups' tiles
};

// An upper bound of the tiles of `rows` rows each (the rows behind the last group count as one more group).
inline int row_tile_count(int R, int E, int rows) {
  const int64_t groups = (int64_t)E + 1 < R ? (int64_t)E + 1 : R;
  return (int)(R / rows + groups);
}

// 64 groups' tiles at a time, summed along the wave; every wave does it for itself (two loads and a dozen exchanges for
// up to 63 groups).
struct RowTileScan {
  int lo, hi, mine, scan;
  __device__ __forceinline__ void step(const int32_t *__restrict__ offsets, int E, int R, int rows, int e0) {
    const int lane = threadIdx.x & 63, e = e0 + lane;
    lo = e <= E ? clamp_offset(offsets, e, R) : R;
    hi = e < E ? max(lo, clamp_offset(offsets, e + 1, R)) : R;
    mine = (hi - lo + rows - 1) / rows;
    scan = mine;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
      const int o = __shfl_up(scan, d);
      if (lane >= d) scan += o;
    }
  }
  __device__ __forceinline__ int total() const { return __builtin_amdgcn_readfirstlane(__shfl(scan, 63)); }
};

// Which of the tiles x columns blocks a workgroup computes.  The chip's eight XCDs take workgroups in turn (number % 8)
// and each has an L2 of its own: an XCD gets a contiguous share of the blocks, in bands of BAND row tiles that walk
// through the column tiles together, so that a band's rows and the weights of a few column tiles stay in its L2.  The
// shares are of the blocks that exist: the launch's bound counts a partial tile for every group.
constexpr int BAND = 4;
__device__ __forceinline__ RowTile find_row_tile(const int32_t *__restrict__ offsets, int E, int R, int rows, int columns,
                                                 int workgroup, int *column) {
  RowTileScan s;
  s.step(offsets, E, R, rows, 0);
  int tiles = s.total();
  if (E >= 64)
    for (int e0 = 64; e0 <= E; e0 += 64) {
      RowTileScan more;
      more.step(offsets, E, R, rows, e0);
      tiles += more.total();
    }
  RowTile t{-1, 0, 0, 0};
  // (bad offsets can make the groups overlap: more tiles than the launch has workgroups for, the rest is left out)
  const int64_t blocks = (int64_t)tiles * columns, share = (blocks + 7) / 8;
  const int64_t block = (workgroup & 7) * share + (workgroup >> 3);
  if ((workgroup >> 3) >= share || block >= blocks) return t;
  const int band = (int)(block / ((int64_t)BAND * columns)), in_band = (int)(block % ((int64_t)BAND * columns));
  const int tall = min(BAND, tiles - band * BAND);
  const int tile = band * BAND + in_band % tall;
  *column = in_band / tall;
  int before = 0;
  for (int e0 = 0; e0 <= E; e0 += 64) {
    if (E >= 64) s.step(offsets, E, R, rows, e0);
    const unsigned long long past = __ballot(before + s.scan > tile);
    if (past) {
      const int f = __ffsll((long long)past) - 1;
      const int first = __builtin_amdgcn_readfirstlane(__shfl(before + s.scan - s.mine, f));
      const int glo = __builtin_amdgcn_readfirstlane(__shfl(s.lo, f)), ghi = __builtin_amdgcn_readfirstlane(__shfl(s.hi, f));
      t.expert = e0 + f, t.number = tile;
      t.begin = glo + (tile - first) * rows;
      t.end = min(t.begin + rows, ghi);
      return t;
    }
    before += s.total();
  }
  return t;
}
// The expert with the n-th most rows (up to 64 experts; otherwise n itself): work that is unequal from expert to expert is
// handed out largest first, so that no large piece is left for the end.
__device__ __forceinline__ int largest_first(const int32_t *__restrict__ offsets, int E, int R, int n) {
  if (E > 64) return n;
  const int lane = threadIdx.x & 63;
  const int lo = lane < E ? clamp_offset(offsets, lane, R) : 0, hi = lane < E ? max(lo, clamp_offset(offsets, lane + 1, R)) : -1;
  const int mine = hi - lo;  // (-1 behind the last expert)
  int rank = 0;
  for (int e = 0; e < E; ++e) {
    const int other = __builtin_amdgcn_readlane(mine, e);
    rank += other > mine || (other == mine && e < lane);
  }
  const unsigned long long it = __ballot(lane < E && rank == n);
  return it ? __ffsll((long long)it) - 1 : n;
}
// workgroups for up to `tiles` x `columns` blocks: every XCD's share rounded up
inline int64_t row_tile_workgroups(int64_t tiles, int64_t columns) { return (tiles * columns + 7) / 8 * 8; }

}  // namespace dimo
