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
};

// An upper bound of the tiles of `rows` rows each (the rows behind the last group count as one more group).  HALVES: w whole
// tiles and h halves have 2 w + h <= 2 R / rows + groups and h <= 2 groups, so w + h <= R / rows + 3/2 groups.
template <bool HALVES = false>
inline int row_tile_count(int R, int E, int rows) {
  const int64_t groups = (int64_t)E + 1 < R ? (int64_t)E + 1 : R;
  return (int)(R / rows + groups + (HALVES ? groups / 2 + 2 : 0));
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
    sum();
  }
  __device__ __forceinline__ void sum() {
    const int lane = threadIdx.x & 63;
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
//
// HALVES: the rows that do not fill a group's last tile are tiles of rows / 2 (one or two), behind all whole tiles, and
// every XCD has its share of both: a tile of 256 rows has a CU for itself, and a round of partial ones at the end costs as
// much as any (bf16, uneven groups, with halves / without: 16384 rows in 8, 1024 x 1024: 54 / 61 us; in 64: 59 / 64; 65536 in
// 32, 2048 x 2048: 630 / 644; even groups without partial tiles the same).
constexpr int BAND = 4;
// the groups' tiles of the e0-th 64 of them: whole ones or (part 1) halves of what is left
template <bool HALVES>
__device__ __forceinline__ void scan_part(RowTileScan &s, const int32_t *__restrict__ offsets, int E, int R, int rows, int e0,
                                          int part) {
  s.step(offsets, E, R, rows, e0);
  if constexpr (HALVES) {
    const int size = s.hi - s.lo, whole = size / rows;
    s.mine = part ? (size - whole * rows + rows / 2 - 1) / (rows / 2) : whole;
    s.sum();
  }
}
template <bool HALVES>
__device__ __forceinline__ RowTile find_row_tile(const int32_t *__restrict__ offsets, int E, int R, int rows, int columns,
                                                 int workgroup, int *column) {
  RowTile t{-1, 0, 0};
  int at = workgroup >> 3;  // in the XCD's share
  for (int part = 0; part < (HALVES ? 2 : 1); ++part) {
    RowTileScan s;
    scan_part<HALVES>(s, offsets, E, R, rows, 0, part);
    int tiles = s.total();
    if (E >= 64)
      for (int e0 = 64; e0 <= E; e0 += 64) {
        RowTileScan more;
        scan_part<HALVES>(more, offsets, E, R, rows, e0, part);
        tiles += more.total();
      }
    // (bad offsets can make the groups overlap: more tiles than the launch has workgroups for, the rest is left out)
    const int64_t blocks = (int64_t)tiles * columns, share = (blocks + 7) / 8;
    const int64_t block = (workgroup & 7) * share + at;
    if (at >= share) {
      at -= (int)share;
      continue;
    }
    if (block >= blocks) return t;
    const int band = (int)(block / ((int64_t)BAND * columns)), in_band = (int)(block % ((int64_t)BAND * columns));
    const int tall = min(BAND, tiles - band * BAND);
    const int tile = band * BAND + in_band % tall;
    *column = in_band / tall;
    int before = 0;
    for (int e0 = 0; e0 <= E; e0 += 64) {
      if (E >= 64) scan_part<HALVES>(s, offsets, E, R, rows, e0, part);
      const unsigned long long past = __ballot(before + s.scan > tile);
      if (past) {
        const int f = __ffsll((long long)past) - 1;
        const int first = __builtin_amdgcn_readfirstlane(__shfl(before + s.scan - s.mine, f));
        const int glo = __builtin_amdgcn_readfirstlane(__shfl(s.lo, f)), ghi = __builtin_amdgcn_readfirstlane(__shfl(s.hi, f));
        t.expert = e0 + f;
        t.begin = glo + (part ? (ghi - glo) / rows * rows + (tile - first) * (rows / 2) : (tile - first) * rows);
        t.end = min(t.begin + (part ? rows / 2 : rows), ghi);
        return t;
      }
      before += s.total();
    }
    return t;
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
// workgroups for up to `tiles` x `columns` blocks: every XCD's share (HALVES: both its shares) rounded up
template <bool HALVES = false>
inline int64_t row_tile_workgroups(int64_t tiles, int64_t columns) {
  return (tiles * columns + 7) / 8 * 8 + (HALVES ? 16 : 0);
}

}  // namespace dimo
