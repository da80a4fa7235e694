// How the attention kernel's work is cut.  The tiles of all requests stand in one
// row (request b's from first[b] to first[b + 1]); the row is cut into `ranges`
// equal parts, so that one long request keeps every warp as busy as many short
// ones.  A request that lies in one range is finished there; of one that is cut,
// each range leaves a partial result in a place of its own.
#pragma once

#include <cstdint>

#if defined(__CUDACC__)
#define PPB_HD __host__ __device__ __forceinline__
#else
#define PPB_HD inline
#endif

namespace ppb {

struct KvPlan {
  uint32_t tiles = 0;  // of all requests, at most 2^31
  int ranges = 1;      // at most 2^15
  uint32_t each = 0, rest = 0;  // tiles = ranges * each + rest

  // `most` ranges, or fewer so that each has `least` tiles.
  static PPB_HD KvPlan make(uint32_t tiles, int most, int least) {
    const uint32_t want = (tiles + least - 1) / least;
    KvPlan p;
    p.tiles = tiles;
    p.ranges = want < 1 ? 1 : want < static_cast<uint32_t>(most) ? static_cast<int>(want) : most;
    p.each = tiles / p.ranges;
    p.rest = tiles - p.each * p.ranges;
    return p;
  }
  // First tile of range r: r * tiles / ranges, in 32 bits.
  PPB_HD uint32_t begin(int r) const { return r * each + r * rest / ranges; }
  // The range of a tile: the last r with begin(r) <= tile.
  PPB_HD int of(uint32_t tile) const { return static_cast<int>(((tile + 1ull) * ranges - 1) / tiles); }
  // Where range r leaves its part of the request that begins at tile `first`: a
  // range has at most two requests that others share, the one it begins within
  // (or at) and the one it ends within.
  PPB_HD int slot(int r, uint32_t first) const { return 2 * r + (first > begin(r) ? 1 : 0); }
};

}  // namespace ppb
