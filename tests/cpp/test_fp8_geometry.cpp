// Host checks of fp8_geometry.h, built with g++ by tests/test_geometry8.py.
// Prints one line per check and exits non-zero on the first failure.

#include <algorithm>
#include <climits>
#include <cstdio>
#include <cstdlib>
#include <random>

#include "fp8_geometry.h"

using namespace pa;

#define CHECK(cond, ...)                                        \
  do {                                                          \
    if (!(cond)) {                                              \
      std::fprintf(stderr, "FAIL %s:%d: ", __FILE__, __LINE__); \
      std::fprintf(stderr, __VA_ARGS__);                        \
      std::fprintf(stderr, "\n");                               \
      std::exit(1);                                             \
    }                                                           \
  } while (0)

constexpr int64_t kMostKeys = INT32_MAX - 1024;  // of a request, as the launcher bounds it

// Blocks of the 64 tiles whose addresses a wave makes at once, up to the longest
// request: within its keys, and those of the unit's own tiles as they are.
static void tile_blocks() {
  std::mt19937 rng(1);
  for (int64_t len : {int64_t{1}, int64_t{15}, int64_t{16}, int64_t{17}, int64_t{64}, int64_t{65},
                      int64_t{4097}, int64_t{1} << 20, kMostKeys - 5000, kMostKeys - 4096,
                      kMostKeys - 3000, kMostKeys - 1, kMostKeys})
    for (int i = 0; i < 200; ++i) {
      const int64_t lo = i == 0 ? 0 : rng() % len, base = lo & ~15;
      const int64_t last = (len - 1 - base) / kP16WideKeys;  // of the longest unit
      for (int64_t t : {int64_t{0}, last / 2, std::max(last - 70, int64_t{0}),
                        std::max(last - 1, int64_t{0}), last})
        for (int lane = 0; lane < 64; ++lane)
          for (int wave = 0; wave < kP16Waves; ++wave) {
            const int32_t got = f8_tile_block(static_cast<int32_t>(base),
                                              static_cast<int32_t>(t + lane),
                                              static_cast<int32_t>(last), wave,
                                              static_cast<int32_t>(len));
            const int64_t end = (len - 1) & ~int64_t{15};
            CHECK(got >= base && got <= end, "key block %d of [%lld, %lld]", got,
                  (long long)base, (long long)end);
            if (t + lane <= last)
              CHECK(got == std::min(base + kP16WideKeys * (t + lane) + 16 * wave, end),
                    "tile %lld of %lld keys from %lld on: block %d", (long long)(t + lane),
                    (long long)len, (long long)base, got);
          }
    }
  std::printf("tile blocks ok\n");
}

int main() {
  tile_blocks();
  std::printf("ALL OK\n");
  return 0;
}
