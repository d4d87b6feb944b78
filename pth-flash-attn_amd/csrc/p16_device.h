// p16_device.h -- device building blocks that the kernels of p16.h's partition
// share: products of 16-bit operands, LDS reads of columns, barriers.

#pragma once

#include "attn_device.h"
#include "p16.h"

namespace pa {
namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef int16_t i16x4 __attribute__((ext_vector_type(4)));

template <bool kF16>
__device__ __forceinline__ f32x4 mfma16(u32x4 a, u32x4 b, f32x4 c) {
  if constexpr (kF16)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a),
                                                  __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a),
                                                   __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

template <bool kF16>
__device__ __forceinline__ f32x16 mfma32(u32x4 a, u32x4 b, f32x16 c) {
  if constexpr (kF16)
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a),
                                                  __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a),
                                                   __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// sum + the two values of a pair.
template <bool kF16>
__device__ __forceinline__ float add_pair(uint32_t w, float sum) {
  if constexpr (kF16)
    return __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2, w),
                                  (f16x2){static_cast<_Float16>(1.0f), static_cast<_Float16>(1.0f)},
                                  sum, false);
  else
    return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, w),
                                           __builtin_bit_cast(bf16x2, 0x3f803f80u), sum, false);
}

// A barrier for LDS alone: __syncthreads also waits for stores to memory.
__device__ __forceinline__ void lds_barrier() {
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// Column l % 16 of four rows of a row-major 16-bit matrix in LDS: lane i of
// each 16 gives the address of row i / 4, columns 4 (i % 4). Without restrict
// the compiler has the read wait for every load to LDS in flight, the next
// tile's.
__device__ __forceinline__ u32x2 column4(const char* __restrict__ a) {
  return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                       (i16x4 __attribute__((address_space(3)))*)(
                                           const_cast<char*>(a))));
}

}  // namespace
}  // namespace pa
