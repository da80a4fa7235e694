// The attention kernel's cut of its work (csrc/kv_plan.h): every tile in one
// range, every partial result in a place of its own within the workspace, and
// the join looks in exactly the places that were written.
#include <cstdio>
#include <cstdlib>
#include <random>
#include <set>
#include <vector>

#include "kv_plan.h"

using ppb::FastDiv;
using ppb::KvPlan;

#define CHECK(x)                                                     \
  do {                                                               \
    if (!(x)) {                                                      \
      std::printf("failed at line %d: %s\n", __LINE__, #x);          \
      std::exit(1);                                                  \
    }                                                                \
  } while (0)

static void check(const std::vector<uint32_t>& tiles, int most) {
  std::vector<uint32_t> first{0};
  for (uint32_t t : tiles) first.push_back(first.back() + t);
  const KvPlan p = KvPlan::make(first.back(), FastDiv::make(most));
  CHECK(p.ranges <= most);
  if (p.tiles == 0) return;
  CHECK(p.ranges >= 1);
  CHECK(p.begin(0) == 0 && p.begin(p.ranges) == p.tiles);
  std::set<std::pair<size_t, int>> written;  // (request, slot)
  std::set<int> slots;
  size_t b = 0;
  for (int r = 0; r < p.ranges; ++r) {
    const uint32_t lo = p.begin(r), hi = p.begin(r + 1);
    CHECK(lo < hi);  // ranges are never more than tiles
    CHECK(p.of(lo) == r && p.of(hi - 1) == r);
    while (first[b + 1] <= lo) ++b;
    for (size_t c = b; c < tiles.size() && first[c] < hi; ++c) {
      if (tiles[c] == 0 || (first[c] >= lo && first[c + 1] <= hi)) continue;
      const int s = p.slot(r, first[c]);
      CHECK(s >= 0 && s < 2 * most);
      CHECK(slots.insert(s).second);
      written.insert({c, s});
    }
  }
  size_t read = 0;
  for (size_t c = 0; c < tiles.size(); ++c) {
    if (tiles[c] == 0) continue;
    const int r0 = p.of(first[c]), r1 = p.of(first[c + 1] - 1);
    if (r0 == r1) continue;
    for (int r = r0; r <= r1; ++r, ++read) CHECK(written.count({c, p.slot(r, first[c])}) == 1);
  }
  CHECK(read == written.size());
}

int main() {
  std::mt19937 rng(1);
  for (int i = 0; i < 4000; ++i) {
    std::vector<uint32_t> t(1 + rng() % (i % 4 ? 20 : 900));
    for (auto& v : t) v = rng() % 3 == 0 ? 0 : 1 + rng() % (1 << rng() % 14);
    check(t, 1 + static_cast<int>(rng() % 1200));
  }
  check({(1u << 31) - 1}, 1184);
  check({1, (1u << 31) - 3, 1}, 1184);
  check({(1u << 31) - 1}, 32767);
  for (int i = 0; i < 2000000; ++i) {
    const uint32_t d = 1 + rng() % (i % 3 ? 70000u : 0x7fffffffu), n = rng() % 0x80000000u;
    const FastDiv f = FastDiv::make(d);
    CHECK(f.quotient(n) == n / d && f.quotient(n / d * d) == n / d && (n < d || f.quotient(n / d * d - 1) == n / d - 1));
    CHECK(f.quotient(0x7fffffffu) == 0x7fffffffu / d);
  }
  check({0, 0, 1, 0}, 148);
  check({0}, 148);
  std::printf("kv_plan_test: ok\n");
}
