// p16_geometry.h -- integer geometry of attention over a paged 16-bit cache
// that the kernels share with the CPU tests (tests/cpp/test_p16_geometry.cpp,
// built by g++).

#pragma once

#include "attn_geometry.h"

namespace pa {

// A request's query tokens: `count` from `first` on.
struct P16Tokens {
  int32_t first, count;
};

// They are [q0, q1) where the starts are in order and within the num_tokens
// that there are. Any others are brought there before they are subtracted: a
// start far below 0 would otherwise wrap to a count of tokens that q and out
// do not have.
PA_HD P16Tokens p16_tokens(int32_t q0, int32_t q1, int32_t num_tokens) {
  const int32_t first = q0 < 0 ? 0 : q0 < num_tokens ? q0 : num_tokens;
  const int32_t last = q1 < first ? first : q1 < num_tokens ? q1 : num_tokens;
  return {first, last - first};
}

}  // namespace pa
