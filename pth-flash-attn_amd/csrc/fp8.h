// fp8.h -- a paged cache in 8-bit floating point with a scale for each block
// of 16 slots and KV head, and rotary positions: what their kernels share, and
// the host launchers.
//
// A value is a code of 8 bits (OCP e4m3: 3 bits of mantissa, 2^-9 to 448) times
// its block's scale 2^(e - 127), held as the byte e. A scale that is a power of
// two costs a floating code nothing: its step is the same share of the value in
// every binade, so all that another scale could gain is part of a binade at the
// small end of a range of 17. It makes every product with the scale exact, a
// block that grows exact but for its smallest codes, and suits the
// conversions of the hardware, which take a scale's exponent.

#pragma once

#include <string>

#include "p16.h"

namespace pa {

constexpr int kF8Span = 16;     // slots of a scale
constexpr int kF8MostExp = 246; // of a scale: 448 x 2^119 is the largest value

// Host side.
constexpr int64_t kMostThreads = 0xffffffff;  // of a launch
int32_t launch_rotary(const PthAttnRotaryArgs& a, hipStream_t stream);
int32_t launch_write_f8(const PthAttnWriteF8Args& a, hipStream_t stream);
int32_t launch_gather_f8(const PthAttnGatherF8Args& a, hipStream_t stream);
int32_t launch_paged_f8(const PthAttnPagedF8Args& a, hipStream_t stream);
hipError_t launch_f8_rows_kernel(const F8Params& p, bool f16, int head_size, hipStream_t stream);
hipError_t launch_f8_wide_kernel(const F8Params& p, bool f16, int head_size, hipStream_t stream);

// A stride of a dimension of n elements, as far as it is used.
inline int64_t used_stride(int64_t stride, int64_t n) { return n > 1 ? stride : 0; }
// Checks of a cache's sizes and, with its data, addresses. "" or what is wrong.
std::string f8_cache_sizes(const PthAttnCacheF8& c);
std::string f8_cache_rows(const PthAttnCacheF8& c);

}  // namespace pa
