// Host-only test of how an XCD's tiles go to workgroups (TilesAtOnce, XcdPlaceOf
// and XcdWorkgroups of kernels/launch_geometry.h, by which the host counts a
// launch's workgroups and the device finds a workgroup's tile): whatever the
// number of CUs and tiles, every tile is made by one workgroup or by four, one
// to each quarter, and nothing else is.
#include <cstdint>
#include <cstdio>
#include <vector>

#include "kernels/launch_geometry.h"

static int g_failures = 0;
#define EXPECT(cond)                                                          \
  do {                                                                        \
    if (!(cond)) {                                                            \
      std::fprintf(stderr, "%s:%d: EXPECT failed: %s\n", __FILE__, __LINE__, #cond); \
      ++g_failures;                                                           \
    }                                                                         \
  } while (0)

// An XCD's `tiles` tiles by `workgroups` workgroups.
static void CheckCover(int at_once, int64_t tiles, int64_t workgroups) {
  std::vector<int> whole(tiles), quarters(tiles);
  for (int64_t place = 0; place < workgroups; ++place) {
    const ruyamd::XcdPlace p = ruyamd::XcdPlaceOf(place, tiles, at_once);
    EXPECT(p.quarter >= -1 && p.quarter <= 3 && p.tile >= 0);
    if (p.tile >= tiles) continue;  // (no tile: the workgroup ends)
    if (p.quarter < 0)
      ++whole[p.tile];
    else
      quarters[p.tile] += 1 << (4 * p.quarter);
  }
  int64_t in_quarters = 0;
  for (int64_t t = 0; t < tiles; ++t) {
    EXPECT((whole[t] == 1 && quarters[t] == 0) || (whole[t] == 0 && quarters[t] == 0x1111));
    in_quarters += whole[t] == 0;
  }
  // Quarters: what is left after full rounds, a quarter of a round at most.
  const int64_t rest = tiles % at_once;
  EXPECT(in_quarters == (tiles >= at_once && rest * 4 <= at_once ? rest : 0));
}

int main() {
  // (Devices and partitions of them, of fewer CUs than XCDs too.)
  for (int compute_units : {1, 2, 3, 7, 8, 9, 15, 16, 31, 32, 38, 64, 80, 128, 252, 256, 304}) {
    const int at_once = ruyamd::TilesAtOnce(compute_units);
    EXPECT(at_once >= 1 && (compute_units < 8 || at_once == compute_units / 8));
    for (int64_t tiles = 0; tiles <= 4 * at_once + 3; ++tiles) {
      CheckCover(at_once, tiles, ruyamd::XcdWorkgroups(tiles, at_once, false));
      // Where the host knows no more than that there are so many tiles at most.
      const int64_t most = ruyamd::XcdWorkgroups(tiles, at_once, true);
      EXPECT(most <= tiles + 3 * (at_once / 4));
      for (int64_t fewer = 0; fewer <= tiles; ++fewer) CheckCover(at_once, fewer, most);
    }
    if (g_failures) break;
  }
  if (g_failures) {
    std::fprintf(stderr, "tile_quarters_test: %d failure(s)\n", g_failures);
    return 1;
  }
  std::printf("tile_quarters_test: all passed\n");
  return 0;
}
