// p16_writer.hip -- keys and values into a paged cache of the model's own
// 16-bit type: a copy of each (token, KV head) row of D values to its slot, or
// one rounding to nearest even of an fp32 row. A lane moves eight values of a
// row of K and of V: one 16-byte load (two of fp32) and one 16-byte store
// each. Rows of the source that are not on 16-byte addresses are read value by
// value.
//
// Bound: HBM. 16,384 tokens of 8 heads of 128 from fp32 (201 MB): 40.5 us, 4.97
// TB/s, a large copy's rate (4.91). 64 tokens of bf16: 2.6 us, a launch.

#include <hip/hip_runtime.h>

#include <string>

#include "attn_device.h"
#include "p16.h"

namespace pa {
namespace {

struct Write16Params {
  const char* key;
  const char* value;
  int64_t s_k_tok, s_k_head, s_v_tok, s_v_head;
  const int64_t* slot_mapping;
  CacheStream k, v;
  int64_t num_slots, block_size;
  int64_t items;  // (token, head) pairs
  Div32 bs_div, heads_div;
  int32_t num_kv_heads;
};

// Eight values of a source row as the cache holds them. kF32: fp32 values;
// kWide: on a 16-byte address.
template <bool kF16, bool kF32, bool kWide>
__device__ __forceinline__ u32x4 eight(const char* src) {
  u32x4 r;
  if constexpr (kF32) {
    f32x4 a, b;
    if constexpr (kWide) {
      a = *reinterpret_cast<const f32x4*>(src);
      b = *reinterpret_cast<const f32x4*>(src + 16);
    } else {
      const float* x = reinterpret_cast<const float*>(src);
      a = (f32x4){x[0], x[1], x[2], x[3]};
      b = (f32x4){x[4], x[5], x[6], x[7]};
    }
    r = (u32x4){pack16<kF16>(a[0], a[1]), pack16<kF16>(a[2], a[3]), pack16<kF16>(b[0], b[1]),
                pack16<kF16>(b[2], b[3])};
  } else if constexpr (kWide) {
    r = *reinterpret_cast<const u32x4*>(src);
  } else {
    const uint16_t* x = reinterpret_cast<const uint16_t*>(src);
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = x[2 * i] | (static_cast<uint32_t>(x[2 * i + 1]) << 16);
  }
  return r;
}

template <int D, bool kF16, bool kF32, bool kWide>
__global__ __launch_bounds__(256) void write_kv_16bit(const Write16Params w) {
  constexpr int kLanes = D / 8, kElt = kF32 ? 4 : 2;
  const int64_t item = static_cast<int64_t>(blockIdx.x) * (256 / kLanes) + threadIdx.x / kLanes;
  if (item >= w.items) return;
  const int c = threadIdx.x % kLanes;
  const uint32_t tok = w.heads_div.div(static_cast<uint32_t>(item));
  const int64_t head = static_cast<int64_t>(item) - static_cast<int64_t>(tok) * w.num_kv_heads;
  const int64_t slot = w.slot_mapping[tok];
  // The rows are read beside the slot, whether or not it is skipped.
  const u32x4 k = eight<kF16, kF32, kWide>(w.key + static_cast<int64_t>(tok) * w.s_k_tok +
                                           head * w.s_k_head + 8 * kElt * c);
  const u32x4 v = eight<kF16, kF32, kWide>(w.value + static_cast<int64_t>(tok) * w.s_v_tok +
                                           head * w.s_v_head + 8 * kElt * c);
  if (slot < 0 || slot >= w.num_slots) return;
  int64_t page;
  if (w.num_slots < 0x7fffffff) page = w.bs_div.div(static_cast<uint32_t>(slot));
  else page = slot / w.block_size;
  const int64_t in_page = slot - page * w.block_size;
  auto cell = [&](const CacheStream& s) {
    return const_cast<char*>(s.base) + page * s.s_block + in_page * s.s_slot + head * s.s_head +
           16 * c;
  };
  *reinterpret_cast<u32x4*>(cell(w.k)) = k;
  *reinterpret_cast<u32x4*>(cell(w.v)) = v;
}

CacheStream stream_of(const PthAttnStream& s) {
  return CacheStream{static_cast<const char*>(s.data), s.stride_block, s.stride_slot,
                     s.stride_head};
}
// A stride of a dimension of n elements, as far as it is used.
int64_t used(int64_t stride, int64_t n) { return n > 1 ? stride : 0; }
bool on16(const void* p, int64_t a, int64_t b, int64_t c) {
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && a % 16 == 0 && b % 16 == 0 && c % 16 == 0;
}
bool cache_on16(const PthAttnStream& s, const PthAttnWrite16Args& a) {
  return on16(s.data, used(s.stride_block, a.num_blocks), used(s.stride_slot, a.block_size),
              used(s.stride_head, a.num_kv_heads));
}

template <int D>
void write16(const Write16Params& w, bool f16, bool f32, bool wide, hipStream_t stream) {
  constexpr int kPer = 256 / (D / 8);
  const dim3 grid(static_cast<unsigned>((w.items + kPer - 1) / kPer)), block(256);
#define PA_W16(A, B, C) write_kv_16bit<D, A, B, C><<<grid, block, 0, stream>>>(w)
  if (f16) {
    if (f32) wide ? PA_W16(true, true, true) : PA_W16(true, true, false);
    else wide ? PA_W16(true, false, true) : PA_W16(true, false, false);
  } else {
    if (f32) wide ? PA_W16(false, true, true) : PA_W16(false, true, false);
    else wide ? PA_W16(false, false, true) : PA_W16(false, false, false);
  }
#undef PA_W16
}

}  // namespace

int32_t launch_write_kv16(const PthAttnWrite16Args& a, hipStream_t stream) {
  clear_error();
  PA_REQUIRE(a.abi_version == PTH_ATTN_ABI_VERSION,
             "abi_version " + std::to_string(a.abi_version) + " != library ABI " +
                 std::to_string(PTH_ATTN_ABI_VERSION));
  PA_REQUIRE(a.struct_bytes == static_cast<int32_t>(sizeof(PthAttnWrite16Args)),
             "struct_bytes " + std::to_string(a.struct_bytes) + " != sizeof(PthAttnWrite16Args) " +
                 std::to_string(sizeof(PthAttnWrite16Args)));
  PA_REQUIRE(a.head_size == 64 || a.head_size == 128 || a.head_size == 256,
             "head_size must be 64, 128 or 256");
  PA_REQUIRE(a.cache_dtype == PTH_ATTN_F16 || a.cache_dtype == PTH_ATTN_BF16,
             "cache_dtype must be PTH_ATTN_F16 or PTH_ATTN_BF16");
  PA_REQUIRE(a.kv_dtype == a.cache_dtype || a.kv_dtype == PTH_ATTN_F32,
             "kv_dtype must be cache_dtype or PTH_ATTN_F32");
  PA_REQUIRE(a.num_tokens >= 0 && a.num_kv_heads >= 1 && a.block_size >= 1 && a.num_blocks >= 1,
             "num_tokens >= 0, num_kv_heads, block_size and num_blocks >= 1");
  if (a.num_tokens == 0) return PTH_ATTN_OK;
  PA_REQUIRE(a.key && a.value && a.slot_mapping && a.k_cache.data && a.v_cache.data,
             "key, value, slot_mapping and the cache streams must be non-NULL");
  const bool f32 = a.kv_dtype == PTH_ATTN_F32;
  const int64_t elt = f32 ? 4 : 2;
  PA_REQUIRE(reinterpret_cast<uintptr_t>(a.key) % elt == 0 &&
                 reinterpret_cast<uintptr_t>(a.value) % elt == 0 &&
                 a.key_stride_token % elt == 0 && a.key_stride_head % elt == 0 &&
                 a.value_stride_token % elt == 0 && a.value_stride_head % elt == 0,
             "key and value must be aligned to their element");
  PA_REQUIRE(cache_on16(a.k_cache, a) && cache_on16(a.v_cache, a),
             "k_cache and v_cache must have 16-byte aligned rows");
  Write16Params w{};
  w.items = static_cast<int64_t>(a.num_tokens) * a.num_kv_heads;
  // A launch has at most 2^32 threads; one moves eight values.
  PA_REQUIRE(w.items < 0x7fffffff && w.items * (a.head_size / 8) <= 0xffffff00,
             "num_tokens x num_kv_heads must be less than 2^31, its product with head_size "
             "2^35");
  w.key = static_cast<const char*>(a.key);
  w.value = static_cast<const char*>(a.value);
  w.s_k_tok = a.key_stride_token;
  w.s_k_head = a.key_stride_head;
  w.s_v_tok = a.value_stride_token;
  w.s_v_head = a.value_stride_head;
  w.slot_mapping = a.slot_mapping;
  w.k = stream_of(a.k_cache);
  w.v = stream_of(a.v_cache);
  w.num_kv_heads = a.num_kv_heads;
  w.block_size = a.block_size;
  w.num_slots = static_cast<int64_t>(a.num_blocks) * a.block_size;
  w.bs_div = Div32::make(static_cast<uint32_t>(a.block_size));
  w.heads_div = Div32::make(static_cast<uint32_t>(a.num_kv_heads));
  const bool wide = on16(a.key, used(a.key_stride_token, a.num_tokens),
                         used(a.key_stride_head, a.num_kv_heads), 0) &&
                    on16(a.value, used(a.value_stride_token, a.num_tokens),
                         used(a.value_stride_head, a.num_kv_heads), 0);
  const bool f16 = a.cache_dtype == PTH_ATTN_F16;
  switch (a.head_size) {
    case 64: write16<64>(w, f16, f32, wide, stream); break;
    case 256: write16<256>(w, f16, f32, wide, stream); break;
    default: write16<128>(w, f16, f32, wide, stream);
  }
  const hipError_t err = hipGetLastError();
  if (err != hipSuccess)
    return fail(PTH_ATTN_ECUDA,
                std::string("16-bit cache writer launch: ") + hipGetErrorString(err));
  return PTH_ATTN_OK;
}

}  // namespace pa

extern "C" {

int32_t pth_attn_write16_args_bytes(void) {
  return static_cast<int32_t>(sizeof(PthAttnWrite16Args));
}

int32_t pth_attn_write_kv16(const PthAttnWrite16Args* args, void* stream) {
  if (args == nullptr) return pa::fail(PTH_ATTN_EINVAL, "args is NULL");
  return pa::launch_write_kv16(*args, static_cast<hipStream_t>(stream));
}

}  // extern "C"
