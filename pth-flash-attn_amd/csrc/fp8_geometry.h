// fp8_geometry.h -- integer geometry of attention over a paged cache in 8-bit
// floating point that the kernels share with the CPU tests
// (tests/cpp/test_fp8_geometry.cpp, built by g++).

#pragma once

#include "p16_geometry.h"

namespace pa {

// The block of 16 keys that wave `wave` of four brings of 64-key tile t of a
// request's keys from `base` on: the last of its `len` keys' (len > 0) where the
// tile reaches past them. Of a unit whose last tile is `last`, tiles behind that
// are brought to it before they are multiplied: the kernel makes addresses 64
// tiles ahead, and 4,032 keys on from a length near 2^31 wrap to a negative block,
// whose page number is behind the request's row of the block table.
PA_HD int32_t f8_tile_block(int32_t base, int32_t t, int32_t last, int32_t wave, int32_t len) {
  const int32_t at = base + kP16WideKeys * (t < last ? t : last) + 16 * wave;
  const int32_t end = (len - 1) & ~15;
  return at < end ? at : end;
}

}  // namespace pa
