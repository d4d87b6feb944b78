// Host checks of fp8_geometry.h, built with g++ by tests/test_geometry8.py.
// Prints one line per check and exits non-zero on the first failure.

#include <algorithm>
#include <climits>
#include <cmath>
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

constexpr int64_t kMostKeys = kF8MostKeys;

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
                                              static_cast<int32_t>(t + lane), wave,
                                              static_cast<int32_t>(len));
            const int64_t end = (len - 1) & ~int64_t{15};
            CHECK(got >= base && got <= end, "key block %d of [%lld, %lld]", got,
                  (long long)base, (long long)end);
            CHECK(got == std::min(base + kP16WideKeys * (t + lane) + 16 * wave, end),
                  "tile %lld of %lld keys from %lld on: block %d", (long long)(t + lane),
                  (long long)len, (long long)base, got);
          }
    }
  std::printf("tile blocks ok\n");
}

// The shares of a causal request's units: each what its rows see of the request's
// tiles at least, and all together within what the launcher's bound of 2^31 tiles
// counts for them.
struct Request {
  int64_t n, len;  // tokens, keys
  int32_t group, window;
};
static void shares(const Request& q) {
  const int64_t n_rt = (q.n * q.group + kP16WideRows - 1) / kP16WideRows;
  const int64_t lo = std::max<int64_t>(
      (q.window ? std::max<int64_t>(q.len - q.window, 0) : 0) - (q.n - 1), 0);
  const int64_t base = lo & ~15;
  const int64_t n_kt = std::max<int64_t>((q.len - base + 63) / 64, 1);
  const F8Steps s = f8_causal_steps(static_cast<int32_t>(q.n), static_cast<int32_t>(q.len),
                                    static_cast<int32_t>(n_rt), static_cast<int32_t>(n_kt),
                                    q.group, q.window);
  const Div32 div = Div32::make(static_cast<uint32_t>(q.group));
  const auto before = [&](int64_t m) {
    return static_cast<int64_t>(f8_tiles_before(s, static_cast<int32_t>(m), q.group, div));
  };
  // As the launcher: of no request more keys, and of a window no more than its tokens'.
  const int64_t span = q.window ? std::min<int64_t>(q.len, q.window + q.n - 1 + 15) : q.len;
  const int64_t key_tiles = std::max<int64_t>((span + 63) / 64, 1);
  if (n_rt * (key_tiles + 6) > INT32_MAX) return;  // refused
  CHECK(before(0) == 0, "tiles before the first unit");
  CHECK(before(n_rt) <= n_rt * (key_tiles + 6),
        "%lld tokens of %lld keys, G %d, window %d: %lld tiles of %lld units", (long long)q.n,
        (long long)q.len, q.group, q.window, (long long)before(n_rt), (long long)n_rt);
  // All units, of many the first and the last ones and some between.
  const int64_t step = std::max<int64_t>(n_rt / 300, 1);
  for (int64_t u = 0; u < n_rt; u += u < 50 || u > n_rt - 50 ? 1 : step) {
    const auto hi_of = [&](int64_t t) { return std::max<int64_t>(q.len - (q.n - 1 - t), 0); };
    const auto lo_of = [&](int64_t hi) { return q.window ? std::max<int64_t>(hi - q.window, 0) : 0; };
    const int64_t first = hi_of(128 * u / q.group);
    const int64_t last = hi_of(std::min(128 * u + 127, q.n * q.group - 1) / q.group);
    const int64_t from = lo_of(first) > base ? (lo_of(first) - base) / 64 : 0;
    const int64_t to = last > base ? (last - base + 63) / 64 : 0;
    const int64_t have = before(u + 1) - before(u);
    CHECK(have >= 1 && have >= to - from,
          "%lld tokens of %lld keys, G %d, window %d: unit %lld has %lld tiles, needs %lld",
          (long long)q.n, (long long)q.len, q.group, q.window, (long long)u, (long long)have,
          (long long)(to - from));
  }
}
static void unit_shares() {
  std::mt19937 rng(2);
  const auto log = [&](double most) {
    return static_cast<int64_t>(std::exp(std::uniform_real_distribution<>(0.0, std::log(most))(rng)));
  };
  for (int32_t group : {1, 2, 3, 4, 5, 7, 8, 17, 64})
    for (int i = 0; i < 6000; ++i) {
      Request q{log(1 << 20), log(1 << 21), group, 0};
      if (i % 3 == 0) q.len += q.n;             // behind a prefix, as most are
      if (i % 17 == 0) q.len = q.n;             // alone
      if (i % 19 == 0) q.len = q.len & 127;     // more tokens than keys
      if (i % 23 == 0) q.len = 0;
      if (i % 2 == 0) q.window = static_cast<int32_t>(log(1 << 16));
      if (q.window >= q.len) q.window = 0;      // as the launcher
      shares(q);
    }
  for (int64_t n : {4096, 1 << 20, 1 << 24})
    for (int64_t len : {0, 1, 64, 65, 100, 4000, 4095})
      for (int32_t group : {1, 4, 64}) shares({n, len, group, 0});
  std::printf("unit shares ok\n");
}

// A request's keys and a tile of a whole unit, the next power of two, stay below 2^31
// together, whatever the units.
static void whole_units() {
  for (int32_t d : {64, 128, 256})
    for (int32_t cus : {1, 256})
      for (int64_t span : {int64_t{1}, int64_t{1024}, int64_t{5000}, (int64_t{1} << 30) - 1,
                           int64_t{1} << 30, (int64_t{1} << 30) + 1, kMostKeys})
        for (int64_t units : {int64_t{1}, int64_t{256}, int64_t{1} << 20, int64_t{1} << 28}) {
          if (!f8_whole_wide(d, span, units, cus)) continue;
          int64_t tile = 1;
          while (tile < span) tile *= 2;
          CHECK(span + tile - 1 <= INT32_MAX, "units of %lld keys whole", (long long)span);
        }
  CHECK(f8_whole_wide(128, 8192, 2048, 256) && !f8_whole_wide(128, 8192, 64, 256),
        "one prompt of 8,192 tokens, eight heads and one");
  std::printf("whole units ok\n");
}

int main() {
  tile_blocks();
  unit_shares();
  whole_units();
  std::printf("ALL OK\n");
  return 0;
}
