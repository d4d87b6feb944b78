// p16_geometry.h -- integer geometry of attention over a paged 16-bit cache
// that the kernels share with the CPU tests (tests/cpp/test_p16_geometry.cpp,
// built by g++).

#pragma once

#include "attn_geometry.h"

namespace pa {

// Row tiles of the two kernels, and the wide one's key tile (the other's is 32
// for each wave of a unit).
constexpr int kP16Waves = 4;
constexpr int kP16RowsRows = 16;
constexpr int kP16WideRows = 32 * kP16Waves, kP16WideKeys = 64;

// Work-groups of either attention kernel that a compute unit holds, by their
// registers, and so the most whose slots are in use where groups are cut.
PA_HD constexpr int32_t p16_resident(int32_t head_size) {
  return head_size == 64 ? 3 : head_size == 128 ? 2 : 1;
}

// Workspace: two slots of each such work-group, of the most rows that a slot of
// either kernel has, D sums with a maximum and a sum to each row; behind them
// the notes (P16Cut), one for each work-group and one before them.
constexpr int32_t kP16NoteWords = 32;  // of a compute unit
inline int64_t p16_workspace_floats(int32_t head_size, int32_t cus) {
  const int64_t rows = int64_t{2} * p16_resident(head_size) * kP16WideRows;
  return cus * (rows * (head_size + 2) + kP16NoteWords);
}

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
