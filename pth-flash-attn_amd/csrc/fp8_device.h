// fp8_device.h -- device building blocks of a cache in 8-bit floating point
// (fp8.h): scales, conversions of codes.

#pragma once

#include "fp8.h"
#include "p16_device.h"

namespace pa {
namespace {

// A run of codes, and its words.
template <int kWords>
struct Words;
template <>
struct Words<1> { typedef uint32_t type; };
template <>
struct Words<2> { typedef u32x2 type; };
template <>
struct Words<4> { typedef u32x4 type; };
__device__ __forceinline__ uint32_t word(uint32_t w, int) { return w; }
template <class V>
__device__ __forceinline__ uint32_t word(const V& w, int i) { return w[i]; }

// 2^(e - 127), 0 for e = 0.
__device__ __forceinline__ float f8_scale(uint32_t e) {
  return __builtin_bit_cast(float, min(e, static_cast<uint32_t>(kF8MostExp)) << 23);
}

// Where a block of 16 keys begins in K and in V, and its exponents (K's, and V's
// above bit 8). The lanes of a wave make these for 64 blocks at once, kept in LDS or
// in registers: page numbers, products of strides and scales worked out block by
// block on the scalar unit are some 100 instructions each.
struct F8Block {
  uint64_t k, v;
  uint32_t e;
};
// The block of the keys from `kb` on: a multiple of 16, within the table.
__device__ __forceinline__ F8Block f8_block(const F8Params& p, const int32_t* table, int32_t head,
                                            int32_t kb) {
  const uint32_t page = mulhi32(static_cast<uint32_t>(kb), p.bs_div.mul) >> p.bs_div.shift;
  const int32_t entry = table[page];
  const int64_t id =
      static_cast<uint32_t>(entry) < static_cast<uint32_t>(p.num_blocks) ? entry : 0;
  const int32_t in = kb - static_cast<int32_t>(page * p.bs_div.d);
  F8Block b;
  b.k = reinterpret_cast<uint64_t>(p.k.base + head * p.k.s_head) + id * p.k.s_block +
        static_cast<uint64_t>(in) * static_cast<uint32_t>(p.k.s_slot);
  b.v = reinterpret_cast<uint64_t>(p.v.base + head * p.v.s_head) + id * p.v.s_block +
        static_cast<uint64_t>(in) * static_cast<uint32_t>(p.v.s_slot);
  const int64_t e = (id * p.n_sub + in / kF8Span) * p.num_kv_heads + head;
  b.e = static_cast<uint32_t>(p.k_exp[e]) | static_cast<uint32_t>(p.v_exp[e]) << 8;
  return b;
}
// A wave's blocks in LDS.
struct F8Window {
  u32x4 address[64];  // of K, of V
  uint32_t e[64];
};
// An address in memory made of its words, which are the same in all lanes. (Of no
// named address space, its loads would count and wait with those from LDS.)
typedef const char __attribute__((address_space(1))) * GlobalBytes;
__device__ __forceinline__ GlobalBytes f8_uniform(uint32_t lo, uint32_t hi) {
  return reinterpret_cast<GlobalBytes>(
      static_cast<uint64_t>(static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(lo))) |
      static_cast<uint64_t>(static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(hi))) << 32);
}

// Two codes of a word (its low or high half) as two 16-bit values, scaled.
template <bool kF16>
__device__ __forceinline__ uint32_t f8_pair_lo(uint32_t w, float scale) {
  if constexpr (kF16)
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, scale, false));
  else
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, false));
}
template <bool kF16>
__device__ __forceinline__ uint32_t f8_pair_hi(uint32_t w, float scale) {
  if constexpr (kF16)
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, scale, true));
  else
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, true));
}
// Eight codes as eight 16-bit values.
template <bool kF16>
__device__ __forceinline__ u32x4 f8_eight(uint32_t a, uint32_t b, float scale) {
  return (u32x4){f8_pair_lo<kF16>(a, scale), f8_pair_hi<kF16>(a, scale), f8_pair_lo<kF16>(b, scale),
                 f8_pair_hi<kF16>(b, scale)};
}
// 0x80 in each byte of a word that is a NaN code (0x7f or 0xff).
__device__ __forceinline__ uint32_t f8_nan_bytes(uint32_t w) {
  return ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
}
// Whether a word holds one.
__device__ __forceinline__ bool f8_has_nan(uint32_t w) {
  return f8_nan_bytes(w) != 0;
}
// Two bf16 values, 0 for a NaN.
__device__ __forceinline__ uint32_t f8_without_nan(uint32_t w) {
  return ((w & 0x7fffu) > 0x7f80u ? 0u : w & 0xffffu) |
         ((w & 0x7fff0000u) > 0x7f800000u ? 0u : w & 0xffff0000u);
}

}  // namespace
}  // namespace pa
