// Rows in segments of uneven lengths (samples of a batch, groups of an expert layer), cut into tiles that do not cross a
// segment's end.  The ends are on the device only: a launch has workgroups for the most tiles there can be, and each
// finds its own from the starts.
#ifndef MLUOP_AMD_CORE_RAGGED_H_
#define MLUOP_AMD_CORE_RAGGED_H_

#include <hip/hip_runtime.h>

#include <cstdint>

#include "core/wave_scan.h"

namespace mluop {

struct RaggedTile {
  int segment;      // -1: there is no such tile
  int first, rows;  // of the tile
  int in_segment;   // the tile's number within its segment
  int segment_first, segment_rows;
};

// Rows of segment s of [0, segments), inside [0, rows) whatever the starts hold; starts null: one segment of all rows.
__device__ __forceinline__ void segmentRows(const int32_t *starts, int rows, int s, int *first, int *count) {
  if (starts == nullptr) {
    *first = 0;
    *count = rows;
    return;
  }
  const int a = starts[s], b = starts[s + 1];
  const int lo = a < 0 ? 0 : (a > rows ? rows : a), hi = b < lo ? lo : (b > rows ? rows : b);
  *first = lo;
  *count = hi - lo;
}

// The same with what lies outside of all segments: 0 the rows in front of the first, segments + 1 those behind the last,
// s the rows of segment s - 1.
__device__ __forceinline__ void segmentOrOutside(const int32_t *starts, int rows, int segments, int s, int *first,
                                                 int *count) {
  if (s > 0 && s <= segments) {
    segmentRows(starts, rows, s - 1, first, count);
    return;
  }
  *first = *count = 0;
  if (starts == nullptr) return;
  const int edge = starts[s == 0 ? 0 : segments];
  const int at = edge < 0 ? 0 : (edge > rows ? rows : edge);
  if (s == 0) {
    *count = at;
  } else {
    *first = at;
    *count = rows - at;
  }
}

// Most tiles of `tile_rows` rows that `rows` rows in `segments` segments can make.
inline int64_t mostRaggedTiles(int64_t rows, int64_t segments, int64_t tile_rows) {
  const int64_t filled = rows < segments ? rows : segments;
  return rows / tile_rows + filled;
}

// Tile `tile` of all tiles of tile_rows rows, segment after segment.  By whole waves; the answer is the same in all
// lanes.  64 segments at a time: a load, a scan and a ballot.  OUTSIDE: the segments are those of segmentOrOutside.
template <bool OUTSIDE>
__device__ __forceinline__ RaggedTile findRaggedTile(const int32_t *starts, int rows, int segments, int tile_rows,
                                                     int tile) {
  const int lane = threadIdx.x & 63;
  RaggedTile t;
  t.segment = -1;
  t.first = t.rows = t.in_segment = t.segment_first = t.segment_rows = 0;
  int before = 0;
  const int all = OUTSIDE ? segments + 2 : segments;
  for (int base = 0; base < all; base += 64) {
    int first = 0, count = 0;
    if (base + lane < all) {
      if (OUTSIDE)
        segmentOrOutside(starts, rows, segments, base + lane, &first, &count);
      else
        segmentRows(starts, rows, base + lane, &first, &count);
    }
    const int tiles = (count + tile_rows - 1) / tile_rows;
    const int upto = before + waveInclusiveScan(tiles);
    const unsigned long long behind = __ballot(tile < upto);
    if (behind != 0) {
      const int l = __ffsll((long long)behind) - 1;
      t.segment_first = __builtin_amdgcn_readlane(first, l);
      t.segment_rows = __builtin_amdgcn_readlane(count, l);
      t.in_segment = tile - __builtin_amdgcn_readlane(upto - tiles, l);
      // (starts that overlap can add up to more than an int holds)
      if ((uint32_t)t.in_segment >= (uint32_t)__builtin_amdgcn_readlane(tiles, l)) return t;
      t.segment = base + l;
      t.first = t.segment_first + t.in_segment * tile_rows;
      t.rows = t.segment_rows - t.in_segment * tile_rows;
      if (t.rows > tile_rows) t.rows = tile_rows;
      return t;
    }
    before = __builtin_amdgcn_readlane(upto, 63);
  }
  return t;
}

// All tiles of all segments (OUTSIDE: of segmentOrOutside).
template <bool OUTSIDE>
__device__ __forceinline__ int raggedTiles(const int32_t *starts, int rows, int segments, int tile_rows) {
  const int lane = threadIdx.x & 63;
  const int all = OUTSIDE ? segments + 2 : segments;
  int sum = 0;
  for (int base = 0; base < all; base += 64) {
    int first = 0, count = 0;
    if (base + lane < all) {
      if (OUTSIDE)
        segmentOrOutside(starts, rows, segments, base + lane, &first, &count);
      else
        segmentRows(starts, rows, base + lane, &first, &count);
    }
    sum += __builtin_amdgcn_readlane(waveInclusiveScan((count + tile_rows - 1) / tile_rows), 63);
  }
  return sum;
}

// The tiles of segment `segment`: how many, and the number of the first among all tiles.  Inside [0, most], the tiles that
// mostRaggedTiles says there can be, whatever the starts hold.
__device__ __forceinline__ int raggedTilesOf(const int32_t *starts, int rows, int segment, int tile_rows, int most,
                                             int *first_tile, int *segment_rows) {
  const int lane = threadIdx.x & 63;
  int before = 0;
  for (int base = 0; base < segment; base += 64) {
    int first = 0, count = 0;
    if (base + lane < segment) segmentRows(starts, rows, base + lane, &first, &count);
    const int tiles = (count + tile_rows - 1) / tile_rows;
    before += __builtin_amdgcn_readlane(waveInclusiveScan(tiles), 63);
  }
  int first;
  segmentRows(starts, rows, segment, &first, segment_rows);
  const int tiles = (*segment_rows + tile_rows - 1) / tile_rows;
  *first_tile = before < 0 ? 0 : (before > most ? most : before);
  return tiles < most - *first_tile ? tiles : most - *first_tile;
}

}  // namespace mluop

#endif  // MLUOP_AMD_CORE_RAGGED_H_
