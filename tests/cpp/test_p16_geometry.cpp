// Host checks of p16_geometry.h, built with g++ by tests/test_geometry16.py.
// Prints one line per check and exits non-zero on the first failure.

#include <algorithm>
#include <climits>
#include <cstdio>
#include <cstdlib>
#include <random>
#include <vector>

#include "p16_geometry.h"

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

// Starts of any value give tokens that exist, and [q0, q1) where that is a
// range of them.
static void tokens() {
  const int32_t lo = INT_MIN, hi = INT_MAX;
  std::vector<int32_t> at = {lo, lo + 1, lo + 199, lo + 200, lo + 201, -3, -1, 0, 1, 2, 199,
                             200, 201, 1 << 30, hi - 1, hi};
  std::mt19937 rng(1);
  for (int i = 0; i < 200; ++i) at.push_back(static_cast<int32_t>(rng()));
  for (int32_t n : {0, 1, 200, 1 << 20, hi - 1024})
    for (int32_t q0 : at)
      for (int32_t q1 : at) {
        const P16Tokens t = p16_tokens(q0, q1, n);
        const int64_t first = std::clamp<int64_t>(q0, 0, n);
        const int64_t last = std::clamp<int64_t>(q1, first, n);
        CHECK(t.first == first && t.count == last - first, "starts %d, %d of %d: %d from %d on",
              q0, q1, n, t.count, t.first);
      }
  std::printf("tokens ok\n");
}

// The workspace holds the slots and notes of as many work-groups as a device
// has resident, for any team and rows of a unit, and no more than the largest
// of these takes.
static void workspace() {
  for (int32_t d : {64, 128, 256})
    for (int32_t cus : {1, 256, 304}) {
      const int64_t have = p16_workspace_floats(d, cus);
      int64_t most = 0;
      const int64_t wgs = int64_t{cus} * p16_resident(d);
      for (int64_t rows : {1, 5, kP16RowsRows, 2 * kP16RowsRows, 4 * kP16RowsRows, kP16WideRows})
        most = std::max(most, 2 * wgs * rows * (d + 2));
      CHECK(most + 4 * (wgs + 1) <= have, "D %d: %lld of %lld", d, (long long)most,
            (long long)have);
      CHECK(have - most <= kP16NoteWords * cus, "D %d: %lld floats unused", d,
            (long long)(have - most));
      std::printf("workspace %d %d %lld\n", d, cus, (long long)have);
    }
}

int main() {
  tokens();
  workspace();
  std::printf("ALL OK\n");
  return 0;
}
