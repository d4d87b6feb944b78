// fp8_geometry.h -- integer geometry of attention over a paged cache in 8-bit
// floating point that the kernels share with the CPU tests
// (tests/cpp/test_fp8_geometry.cpp, built by g++).

#pragma once

#include "p16_geometry.h"

namespace pa {

// The most keys of a request. Key positions stay below 2^31 with what the kernels add to
// them: addresses are made 64 tiles ahead (f8_tile_block: 4,080 keys; a block that wrapped
// would be looked up behind the request's row of the block table), chunks of the 16-row
// kernel's waves two ahead (560). Bringing the tiles to a unit's last one in the kernel
// instead costs 0.2 to 1 % (4 prompts behind prefixes, heads of 128, 723 us for 721).
constexpr int32_t kF8MostKeys = INT32_MAX - 8192;

// The block of 16 keys that wave `wave` of four brings of 64-key tile t of a
// request's keys from `base` on (t at most 63 tiles behind the last): the last of its `len`
// keys' (len > 0) where the tile reaches past them.
PA_HD int32_t f8_tile_block(int32_t base, int32_t t, int32_t wave, int32_t len) {
  const int32_t at = base + kP16WideKeys * t + 16 * wave;
  const int32_t end = (len - 1) & ~15;
  return at < end ? at : end;
}

// Causal 128-row units see a different number of key tiles each: in tokens, unit
// u's last row sees c + (128 u + 127) / G + 1 keys at most, c being the request's
// keys before its tokens. Its share of the stream is an upper bound of that
// whose sums over the units before m have a closed form,
//   F(m) = floor((m G (c + 128) + 64 m (m + 1)) / 64 G),
// within two tiles of the unit's need: F's steps are at least what the sum under
// the floor grows by, less 1, and that leaves the need and the 63 / 64 that it is
// rounded up by. Where a bound C of what any unit sees is less for the units from
// some one on, these have C each: of a window, what it and a unit's tokens cover; of
// tokens without a place among the keys (more tokens than keys), all tiles, beyond
// which F would grow with the square of the tokens. So a request's units have at most
// six tiles each more than its keys.
struct F8Steps {
  int32_t units;   // row tiles
  int32_t linear;  // of these, the first ones that F holds for
  int32_t cap;     // of each behind them
  int32_t before;  // c; -1: `cap` tiles each
};
PA_HD F8Steps f8_causal_steps(int32_t tokens, int32_t len, int32_t n_rt, int32_t n_kt,
                              int32_t group, int32_t window) {
  const int32_t c = len > tokens ? len - tokens : 0;
  F8Steps s = {n_rt, n_rt, n_kt, c};
  if (window > 0) {
    const int32_t per = 128 / group + 2;  // tokens of a unit
    s.cap = ((window + per + 63) >> 6) + 2;
    if (len < tokens && n_kt < s.cap) s.cap = n_kt;
  }
  if (window > 0 || len < tokens) {
    const int64_t from = (64 * static_cast<int64_t>(s.cap) - c - 128) * group >> 7;
    s.linear = from < 0 ? 0 : from < n_rt ? static_cast<int32_t>(from) : n_rt;
  }
  return s;
}
// Tiles of a head's units before m.
PA_HD int32_t f8_tiles_before(const F8Steps& s, int32_t m, int32_t group, const Div32& g_div) {
  if (s.before < 0) return m * s.cap;
  const int64_t l = m < s.linear ? m : s.linear;
  const uint64_t sum =
      static_cast<uint64_t>(l * (static_cast<int64_t>(group) * (s.before + int64_t{128})) +
                            64 * l * (l + 1)) >> 6;
  const uint32_t f = sum >> 31 == 0 ? g_div.div(static_cast<uint32_t>(sum))
                                    : static_cast<uint32_t>(sum / static_cast<uint32_t>(group));
  return static_cast<int32_t>(f) + (m > s.linear ? m - s.linear : 0) * s.cap;
}

// Whether every unit of 128 rows is left whole (one "tile"): where all are short, or as
// many as the longest has a share in the whole. Whole ones end unevenly, cut ones write
// and read their sums. Prompts, 8 heads of 128, whole and cut: 1 of 2,048 tokens 63 and 74
// us, of 8,192 549 and 611; 4 of 2,048 175 and 216; 4 of 1,900 behind 5,900 keys 855 and
// 905; 12 of 100 to 2,000 behind up to 7,000 642 and 723; one head, 1 of 2,048 54 and 40, 1
// of 8,192 208 and 191. Heads of 256, 4 of them: 1 of 1,024 58 and 52, of 4,096 208 and
// 280; 5 of 500 to 2,500 behind 100 to 6,200 440 and 542. Many short units are better
// walked by work-groups that stay: 64 of 256 140 and 122.
inline bool f8_whole_wide(int32_t head_size, int64_t span, int64_t units, int32_t cus) {
  if (span > int64_t{1} << 30) return false;  // such a tile's keys are added to a length
  if (units > 5 * p16_resident(head_size) * cus && span < 1024) return false;
  if (head_size == 256) return span <= 512 || (units >= cus && span * cus <= 2560 * units);
  return span <= 1024 || span * cus <= 1280 * units;
}

}  // namespace pa
