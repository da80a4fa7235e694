// How the attention kernel's work is cut.  The tiles of all requests stand in one
// row (request b's from first[b] to first[b + 1]); the row is cut into equal
// ranges, so that one long request keeps every warp as busy as many short
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

// n / d for n < 2^31 by a product: with 2^(k-1) < d <= 2^k and m = 2^(31+k) / d
// rounded up past it, n m / 2^(31+k) lies above n / d by less than n / 2^(31+k) < 1 / d.
// (The kernels divide by sizes that the host knows; a division by a variable is
// some 30 instructions in a row, and a warp's start had ten of them.)
struct FastDiv {
  uint32_t by = 1, times = 0, shift = 0;

  static FastDiv make(uint32_t d) {
    uint32_t k = 0;
    while ((1ull << k) < d) ++k;
    return {d, static_cast<uint32_t>((1ull << (31 + k)) / d + 1), 31 + k};
  }
  PPB_HD uint32_t quotient(uint32_t n) const { return static_cast<uint32_t>((static_cast<uint64_t>(n) * times) >> shift); }
};

struct KvPlan {
  uint32_t tiles = 0;  // of all requests, below 2^31
  int ranges = 1;      // one for each tile, or `most`, at most 2^15
  uint32_t each = 1, rest = 0;  // tiles = ranges * each + rest
  FastDiv most;

  static PPB_HD KvPlan make(uint32_t tiles, FastDiv most) {
    KvPlan p;
    p.tiles = tiles;
    p.most = most;
    p.ranges = static_cast<int>(tiles < most.by ? tiles : most.by);
    if (tiles >= most.by) {
      p.each = most.quotient(tiles);
      p.rest = tiles - p.each * most.by;
    }
    return p;
  }
  // First tile of range r: r * tiles / ranges, in 32 bits.
  PPB_HD uint32_t begin(int r) const { return r * each + most.quotient(r * rest); }
  // The range of a tile: the last r with begin(r) <= tile.  The guess in fp32 is
  // next to it at most.
  PPB_HD int of(uint32_t tile) const {
    int r = static_cast<int>(static_cast<float>(tile) * (static_cast<float>(ranges) / static_cast<float>(tiles)));
    r = r < ranges ? r : ranges - 1;
    while (begin(r) > tile) --r;
    while (r + 1 < ranges && begin(r + 1) <= tile) ++r;
    return r;
  }
  // Where range r leaves its part of the request that begins at tile `first`: a
  // range has at most two requests that others share, the one it begins within
  // (or at) and the one it ends within.
  PPB_HD int slot(int r, uint32_t first) const { return 2 * r + (first > begin(r) ? 1 : 0); }
};

}  // namespace ppb
