// fp8_writer.hip -- keys and values into a paged cache in 8-bit floating point,
// and back (fp8.h has the format).
//
// The writer. A block's scale depends on all its tokens of the call, which may
// stand anywhere in slot_mapping. A work-group takes a run of tokens, of one KV
// head or of all, puts the blocks of its tokens into a table in LDS, and reads
// the whole of slot_mapping against it: then it knows of each of its blocks the
// first token of the call and the last token of every slot. It takes the blocks
// whose first token is its own, one for each wave at a time, for each head and
// for K and V apart: the rows of up to 16 tokens in registers, their largest
// value over the wave, the scale, the codes. So a value is read once and a code
// written once, whatever the order of the tokens, in one launch and without an
// atomic in memory. Rows that the block holds already are read with them, before it
// is known whether the scale grows, and written only if it does; not where the call
// begins the block.
//
// Bound: its bytes, behind the reading of slot_mapping (8 heads of 128, bf16, cold:
// 16,384 tokens, 101 MB, 23.0 us); latency for a decode step, whose tokens lie in blocks
// of their own (64 tokens 4.8 us).
//
// The reader. A work-group finds the pages of up to 16 rows in LDS, then each thread
// reads four pieces of codes at once and writes each as 16 bytes, a wave of them a
// kilobyte, past the caches (20,480 tokens, 8 heads of 128, bf16: 23.0 us, 30.0 with
// plain stores). Waves take K or V, not lanes: lanes that differ would read the
// launch's parameters from memory (48 us).
// Bound: its bytes (126 MB, 5.5 TB/s); latency for short prefixes (200 tokens of 4
// heads of 64 2.9 us).

#include <hip/hip_runtime.h>

#include <algorithm>
#include <climits>
#include <string>
#include <type_traits>

#include "fp8_device.h"

namespace pa {
namespace {

constexpr int kThreads = 256;
constexpr int kManyThreads = 1024;
constexpr int kWriteTokens = 128;         // of a work-group, at most
constexpr int kTable = 2 * kWriteTokens;  // entries, a power of two
static_assert(kTable <= kThreads, "a thread looks at an entry");
// A work-group has 256 threads, one head and 2 or 4 tokens where that makes no more than
// four work-groups for a compute unit; otherwise kManyThreads threads, one work-group for
// each compute unit at a time (its registers are half of the unit's or more), of 16 tokens
// and some heads or, from kManyTokens tokens on, of up to kWriteTokens tokens and all heads,
// so that few read slot_mapping. 8 heads of 128, bf16, cold: 2,048 tokens 6.2 us against 7.1
// with all heads, 4,096 tokens 9.2 against 9.0.
constexpr int kManyTokens = 4096;
// A filter of blocks, bits: without it 16,384 tokens take 25.7 us, with it 23.1.
constexpr int kFilter = 16384;
// Of slot_mapping that a thread asks for at once (1, 2, 4, 8: 16,384 tokens 24.4, 23.0,
// 23.1, 23.4 us, 64 tokens 4.7, 4.8, 5.0, 5.3).
constexpr int kSlotsAhead = 2;

struct WriteF8Params {
  const char* src[2];  // keys, values
  int64_t s_tok[2], s_head[2];
  CacheStream cache[2];
  uint8_t* scale[2];
  const int64_t* slot_mapping;
  int64_t num_slots;
  Div32 sub_div;  // blocks of a page
  int32_t n_sub;
  int32_t num_kv_heads;
  int32_t num_tokens;
  int32_t tokens, heads;  // of a work-group
};

// Eight values of a source row. kWide: on a 16-byte address.
template <class T>
struct Eight {
  uint32_t w[2 * sizeof(T)];
  __device__ __forceinline__ float operator[](int i) const {
    T x[8];
    __builtin_memcpy(x, w, sizeof(x));
    return static_cast<float>(x[i]);
  }
};
template <class T, bool kWide>
__device__ __forceinline__ Eight<T> load_eight(const char* src) {
  Eight<T> y;
  if constexpr (kWide) {
#pragma unroll
    for (unsigned i = 0; i < sizeof(T) / 2; ++i) {
      const u32x4 v = reinterpret_cast<const u32x4*>(src)[i];
#pragma unroll
      for (int j = 0; j < 4; ++j) y.w[4 * i + j] = v[j];
    }
  } else {
    T x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = reinterpret_cast<const T*>(src)[i];
    __builtin_memcpy(y.w, x, sizeof(x));
  }
  return y;
}

// The smallest exponent whose scale brings the value with these bits (not
// negative, finite) within 448 = 1.75 x 2^8; 0 for 0.
__device__ __forceinline__ uint32_t exponent_for(uint32_t bits) {
  if (bits == 0) return 0;
  const int e = static_cast<int>(bits >> 23) - 8 + ((bits & 0x7fffffu) > 0x600000u);
  return static_cast<uint32_t>(min(max(e, 1), kF8MostExp));
}

// 448 x 2^119, the largest value that the largest scale's codes reach.
constexpr uint32_t kMostBits = 0x7f600000u;

// Four 32-bit values, within the codes' range or NaN, as codes.
__device__ __forceinline__ uint32_t codes4(float a, float b, float c, float d) {
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  w = __builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
  return static_cast<uint32_t>(w);
}

template <int D, class T, bool kWide, int kThreads>
__global__ __launch_bounds__(kThreads) void write_kv_f8(const WriteF8Params p) {
  constexpr int kLanes = D / 8, kRows = 64 / kLanes, kPasses = kF8Span / kRows;
  constexpr int kWaves = kThreads / 64;
  // Whether values that are all finite and small enough have a way of their own (16,384
  // tokens, 8 heads of 128, bf16: 23.1 us, 26.5 without it and with loads in branches): not
  // where a row's registers would go to scratch (4 heads of 256, fp32: 70.8 us, 35.6).
  constexpr bool kTwo = D * sizeof(T) < 1024;
  __shared__ int32_t s_block[kTable], s_first[kTable], s_row[kTable * kF8Span];
  __shared__ int32_t s_list[kTable];
  __shared__ uint32_t s_maybe[kFilter / 32];
  __shared__ int32_t s_count;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int t0 = static_cast<int>(blockIdx.x) * p.tokens;
  const int t1 = min(t0 + p.tokens, p.num_tokens);
  const int head0 = static_cast<int>(blockIdx.y) * p.heads;
  const int heads = min(p.heads, p.num_kv_heads - head0);

  // The run's slots and the first ones of all are asked for before the table is clear.
  int64_t own = -1, slot[kSlotsAhead];
  if (static_cast<int>(threadIdx.x) < t1 - t0) own = p.slot_mapping[t0 + threadIdx.x];
  const auto ask = [&](int base) {
#pragma unroll
    for (int a = 0; a < kSlotsAhead; ++a)
      slot[a] = p.slot_mapping[min(base + kThreads * a + static_cast<int>(threadIdx.x),
                                   p.num_tokens - 1)];
  };
  ask(0);
  if (threadIdx.x < kTable) {
    s_block[threadIdx.x] = -1;
    s_first[threadIdx.x] = INT32_MAX;
  }
#pragma unroll
  for (int i = 0; i < kTable * kF8Span / kThreads; ++i) s_row[kThreads * i + threadIdx.x] = -1;
#pragma unroll
  for (int i = threadIdx.x; i < kFilter / 32; i += kThreads) s_maybe[i] = 0;
  if (threadIdx.x == 0) s_count = 0;
  __syncthreads();
  const auto place = [](int32_t block) { return (block ^ block >> 8) & (kTable - 1); };
  // A bit for each block, shared by few: most tokens of other runs end there.
  const auto filter = [](int64_t of) {
    const uint32_t block = static_cast<uint32_t>(of / kF8Span);
    return (block ^ block >> 14) & (kFilter - 1);
  };
  const auto known = [&](int64_t of) {
    return static_cast<uint64_t>(of) < static_cast<uint64_t>(p.num_slots);
  };
  // At most half of the entries are taken: every search ends at an empty one.
  if (known(own)) {
    const int32_t block = static_cast<int32_t>(own / kF8Span);
    for (int i = place(block);; i = (i + 1) & (kTable - 1)) {
      const int32_t was = atomicCAS(&s_block[i], -1, block);
      if (was == -1 || was == block) break;
    }
    const uint32_t bit = filter(own);
    atomicOr(&s_maybe[bit >> 5], 1u << (bit & 31));
  }
  __syncthreads();
  for (int base = 0; base < p.num_tokens; base += kSlotsAhead * kThreads) {
    int64_t now[kSlotsAhead];
    bool maybe[kSlotsAhead];
#pragma unroll
    for (int a = 0; a < kSlotsAhead; ++a) {
      now[a] = slot[a];
      const uint32_t bit = filter(now[a]);
      maybe[a] = s_maybe[bit >> 5] >> (bit & 31) & 1;
    }
    if (base + kSlotsAhead * kThreads < p.num_tokens) ask(base + kSlotsAhead * kThreads);
#pragma unroll
    for (int a = 0; a < kSlotsAhead; ++a) {
      const int t = base + kThreads * a + static_cast<int>(threadIdx.x);
      if (!maybe[a] || t >= p.num_tokens || !known(now[a])) continue;
      const int32_t block = static_cast<int32_t>(now[a] / kF8Span);
      for (int i = place(block);; i = (i + 1) & (kTable - 1)) {
        const int32_t is = s_block[i];
        if (is == block) {
          atomicMin(&s_first[i], t);
          atomicMax(&s_row[kF8Span * i + static_cast<int>(now[a] % kF8Span)], t);
        }
        if (is == block || is == -1) break;
      }
    }
  }
  __syncthreads();
  if (threadIdx.x < kTable && s_first[threadIdx.x] >= t0 && s_first[threadIdx.x] < t1)
    s_list[atomicAdd(&s_count, 1)] = threadIdx.x;
  __syncthreads();

  const int c = lane % kLanes, r = lane / kLanes;
  const int units = 2 * heads * s_count;
  for (int u = wave; u < units; u += kWaves) {
    const int kv = u & 1;
    const int of = (u >> 1) / heads, head = head0 + (u >> 1) - of * heads;
    const int entry = __builtin_amdgcn_readfirstlane(s_list[of]);
    const int32_t block = __builtin_amdgcn_readfirstlane(s_block[entry]);
    const int32_t page = static_cast<int32_t>(p.sub_div.div(static_cast<uint32_t>(block)));
    const int32_t sub = block - page * p.n_sub;
    uint8_t* exponent = p.scale[kv] + static_cast<int64_t>(block) * p.num_kv_heads + head;
    const uint32_t had = *exponent;
    const CacheStream& s = p.cache[kv];
    // The block, and the lane's place in it.
    char* cell = const_cast<char*>(s.base) + static_cast<int64_t>(page) * s.s_block +
                 static_cast<int64_t>(kF8Span * sub) * s.s_slot +
                 static_cast<int64_t>(head) * s.s_head;
    const uint32_t in_cell = __umul24(r, static_cast<uint32_t>(s.s_slot)) + 8 * c;
    const int32_t* rows = s_row + kF8Span * entry;
    const bool begun = rows[0] >= 0;
    Eight<T> x[kPasses];
    u32x2 held[kPasses];  // what the block's other rows hold, in case its scale grows
#pragma unroll
    for (int i = 0; i < kPasses; ++i) {
      const int32_t token = rows[kRows * i + r];
      const auto load = [&](int32_t t) {
        return load_eight<T, kWide>(p.src[kv] + static_cast<int64_t>(t) * p.s_tok[kv] +
                                    static_cast<int64_t>(head) * p.s_head[kv] + 8 * sizeof(T) * c);
      };
      if constexpr (kTwo) {
        // Where there is none, the first token's row is read, and not used: without a
        // branch the values stay as they are, in half of the registers.
        x[i] = load(max(token, 0));
#pragma unroll
        for (unsigned j = 0; j < 2 * sizeof(T); ++j)
          x[i].w[j] &= static_cast<uint32_t>(~(token >> 31));
      } else {
        x[i] = Eight<T>{};
        if (token >= 0) x[i] = load(token);
      }
      held[i] = (u32x2){0u, 0u};
      if (token < 0 && !begun)
        held[i] = *reinterpret_cast<const u32x2*>(
            cell + static_cast<int64_t>(kRows * i) * s.s_slot + in_cell);
    }
    // Of all values, and where one is not finite or beyond the largest scale's codes, of
    // the finite ones again.
    const auto largest = [&](auto any) {
      uint32_t most = 0;
#pragma unroll
      for (int i = 0; i < kPasses; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const uint32_t b = __builtin_bit_cast(uint32_t, x[i][j]) & 0x7fffffffu;
          most = max(most, decltype(any)::value || b < 0x7f800000u ? b : 0u);
        }
      return static_cast<uint32_t>(
          __builtin_amdgcn_readfirstlane(wave_max32(static_cast<int32_t>(most))));
    };
    uint32_t top = largest(std::bool_constant<kTwo>{});
    const bool plain = kTwo && top <= kMostBits;
    if (kTwo && !plain) top = largest(std::false_type{});
    const uint32_t old = begun ? 0u : min(had, static_cast<uint32_t>(kF8MostExp));
    const uint32_t e = max(old, exponent_for(top));
    const float unit = e ? __builtin_bit_cast(float, (254u - e) << 23) : 0.0f;
    const bool grown = !begun && e > old;
    const float move =
        old && old + 127 > e ? __builtin_bit_cast(float, (old + 127u - e) << 23) : 0.0f;
    // (Choosing between two values, as below, takes 96 registers in fp32 of 256, an if 158.)
    const auto put = [&](auto fine) {
#pragma unroll
      for (int i = 0; i < kPasses; ++i) {
        u32x2* dst = reinterpret_cast<u32x2*>(
            cell + static_cast<int64_t>(kRows * i) * s.s_slot + in_cell);
        if (rows[kRows * i + r] >= 0) {
          float y[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const float v = x[i][j];
            if constexpr (decltype(fine)::value) {
              y[j] = v * unit;
            } else {
              const uint32_t b = __builtin_bit_cast(uint32_t, v) & 0x7fffffffu;
              const float z = fminf(fmaxf(v * unit, -448.0f), 448.0f);
              y[j] = b < 0x7f800000u ? z : __builtin_nanf("");
            }
          }
          *dst = (u32x2){codes4(y[0], y[1], y[2], y[3]), codes4(y[4], y[5], y[6], y[7])};
        } else if (grown) {
          u32x2 y;
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8(held[i][j], false);
            const f32x2 b = __builtin_amdgcn_cvt_pk_f32_fp8(held[i][j], true);
            y[j] = codes4(a[0] * move, a[1] * move, b[0] * move, b[1] * move);
          }
          *dst = y;
        }
      }
    };
    if (plain) put(std::bool_constant<kTwo>{});
    else put(std::false_type{});
    if (lane == 0 && e != had) *exponent = static_cast<uint8_t>(e);
  }
}

struct GatherF8Params {
  char* dst[2];
  int64_t s_tok[2], s_head[2];
  CacheStream cache[2];
  const uint8_t* scale[2];
  const int32_t* block_table;
  int64_t bt_stride;
  const int32_t* starts;
  const int32_t* first;
  int64_t reach;  // tokens that a row of the block table holds
  Div32 bs_div, item_div;
  int32_t n_sub, num_blocks, num_reqs, num_tokens, num_kv_heads;
  int32_t row_items;  // pieces of a row's heads
  int32_t tokens;     // of a work-group
};

constexpr int kGatherTokens = 16;  // of a work-group, at most
constexpr int kPiecesAhead = 4;    // that a thread asks for at once

template <int D, int kType>  // kType: PTH_ATTN_F32, F16 or BF16
__global__ __launch_bounds__(kThreads) void gather_kv_f8(const GatherF8Params p) {
  constexpr int kBytes = kType == PTH_ATTN_F32 ? 4 : 2;
  constexpr int kCodes = 16 / kBytes, kPieces = D / kCodes;  // of a piece; of a head's row
  __shared__ int64_t s_at[2][kGatherTokens], s_e[kGatherTokens];
  const int t0 = static_cast<int>(blockIdx.x) * p.tokens;
  {
    // The last request that begins at or before the row, if it ends behind it: 16 lanes
    // look for a row's, a 16th of the requests that are left at each step.
    const int of = threadIdx.x / 16, j = threadIdx.x % 16, group = threadIdx.x & 48;
    const int t = t0 + of;
    int lo = 0, hi = of < p.tokens ? p.num_reqs : 0;
    while (lo < hi) {
      const int step = (hi - lo + 15) >> 4, at = lo + (j + 1) * step;
      const bool begun = at <= hi && p.starts[at] <= t;
      const int n = __popcll(__ballot(begun) >> group & 0xffff);
      hi = min(hi, lo + (n + 1) * step - 1);
      lo = min(lo + n * step, hi);
    }
    if (j == 0 && of < p.tokens) {
      int64_t e = -2;  // -2: no request's; -1: no page
      int64_t k = 0, v = 0;
      if (t < p.num_tokens && lo < p.num_reqs && p.starts[lo] <= t) {
        e = -1;
        const int64_t pos = static_cast<int64_t>(p.first ? p.first[lo] : 0) + t -
                            static_cast<int64_t>(p.starts[lo]);
        if (pos >= 0 && pos < p.reach) {
          const uint32_t entry = p.bs_div.div(static_cast<uint32_t>(pos));
          const int32_t page = p.block_table[lo * p.bt_stride + entry];
          if (page >= 0 && page < p.num_blocks) {
            const int64_t in = pos - static_cast<int64_t>(entry) * p.bs_div.d;
            k = page * p.cache[0].s_block + in * p.cache[0].s_slot;
            v = page * p.cache[1].s_block + in * p.cache[1].s_slot;
            e = (static_cast<int64_t>(page) * p.n_sub + in / kF8Span) * p.num_kv_heads;
          }
        }
      }
      s_at[0][of] = k;
      s_at[1][of] = v;
      s_e[of] = e;
    }
  }
  __syncthreads();
  // K by the even waves, V by the odd ones.
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), kv = wave & 1;
  const CacheStream s = p.cache[kv];
  const uint8_t* exponents = p.scale[kv];
  char* out = p.dst[kv] + static_cast<int64_t>(t0) * p.s_tok[kv];
  constexpr int kStep = kThreads / 2;
  const int items = p.tokens * p.row_items;
  for (int base = (wave >> 1) * 64 + static_cast<int>(threadIdx.x & 63); base < items;
       base += kPiecesAhead * kStep) {
    typedef typename Words<kCodes / 4>::type Piece;
    Piece w[kPiecesAhead];
    uint32_t exponent[kPiecesAhead];
    char* dst[kPiecesAhead];
#pragma unroll
    for (int a = 0; a < kPiecesAhead; ++a) {
      const int i = min(base + kStep * a, items - 1);
      const int t = static_cast<int>(p.item_div.div(static_cast<uint32_t>(i)));
      const int item = i - t * p.row_items;
      const int head = item / kPieces, c = item % kPieces;
      // Where there is no page, the null page's codes are read, and not used.
      const int64_t e = s_e[t];
      w[a] = *reinterpret_cast<const Piece*>(s.base + s_at[kv][t] + head * s.s_head + kCodes * c);
      exponent[a] = exponents[max(e, int64_t{0}) + head];
      if (e < 0) {
        w[a] = Piece{};
        exponent[a] = 0;
      }
      dst[a] = base + kStep * a < items && e != -2
                   ? out + t * p.s_tok[kv] + head * p.s_head[kv] + kCodes * kBytes * c
                   : nullptr;
    }
#pragma unroll
    for (int a = 0; a < kPiecesAhead; ++a) {
      const float scale = f8_scale(exponent[a]);
      float x[kCodes];
#pragma unroll
      for (int j = 0; j < kCodes / 4; ++j) {
        const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8(word(w[a], j), false);
        const f32x2 hi = __builtin_amdgcn_cvt_pk_f32_fp8(word(w[a], j), true);
        x[4 * j] = lo[0] * scale;
        x[4 * j + 1] = lo[1] * scale;
        x[4 * j + 2] = hi[0] * scale;
        x[4 * j + 3] = hi[1] * scale;
      }
      if (dst[a] == nullptr) continue;
      u32x4 y;
      if constexpr (kType == PTH_ATTN_F32) {
        y = __builtin_bit_cast(u32x4, (f32x4){x[0], x[1], x[2], x[3]});
      } else {
        constexpr bool kF16 = kType == PTH_ATTN_F16;
#pragma unroll
        for (int j = 0; j < 4; ++j) y[j] = pack16<kF16>(x[2 * j], x[2 * j + 1]);
      }
      __builtin_nontemporal_store(y, reinterpret_cast<u32x4*>(dst[a]));
    }
  }
}

CacheStream stream_of(const PthAttnStream& s) {
  return CacheStream{static_cast<const char*>(s.data), s.stride_block, s.stride_slot,
                     s.stride_head};
}
bool on16(const void* p, int64_t tok, int64_t n_tok, int64_t head, int64_t n_head) {
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && used_stride(tok, n_tok) % 16 == 0 &&
         used_stride(head, n_head) % 16 == 0;
}

template <int D, class T, int kThreads>
void write_as(const WriteF8Params& w, bool wide, dim3 grid, hipStream_t stream) {
  if (wide) write_kv_f8<D, T, true, kThreads><<<grid, kThreads, 0, stream>>>(w);
  else write_kv_f8<D, T, false, kThreads><<<grid, kThreads, 0, stream>>>(w);
}
template <int D, class T>
void write_t(const WriteF8Params& w, bool wide, bool many, dim3 grid, hipStream_t stream) {
  if (many) write_as<D, T, kManyThreads>(w, wide, grid, stream);
  else write_as<D, T, kThreads>(w, wide, grid, stream);
}
template <int D>
void write_d(const WriteF8Params& w, int dtype, bool wide, bool many, dim3 grid,
             hipStream_t stream) {
  if (dtype == PTH_ATTN_F32) write_t<D, float>(w, wide, many, grid, stream);
  else if (dtype == PTH_ATTN_F16) write_t<D, _Float16>(w, wide, many, grid, stream);
  else write_t<D, __bf16>(w, wide, many, grid, stream);
}
template <int D>
void gather_d(const GatherF8Params& g, int dtype, dim3 grid, hipStream_t stream) {
  if (dtype == PTH_ATTN_F32) gather_kv_f8<D, PTH_ATTN_F32><<<grid, kThreads, 0, stream>>>(g);
  else if (dtype == PTH_ATTN_F16) gather_kv_f8<D, PTH_ATTN_F16><<<grid, kThreads, 0, stream>>>(g);
  else gather_kv_f8<D, PTH_ATTN_BF16><<<grid, kThreads, 0, stream>>>(g);
}

}  // namespace

std::string f8_cache_sizes(const PthAttnCacheF8& c) {
  if (c.head_size != 64 && c.head_size != 128 && c.head_size != 256)
    return "head_size must be 64, 128 or 256";
  if (c.num_blocks < 1 || c.num_kv_heads < 1 || c.num_kv_heads > 65535)
    return "num_blocks >= 1, num_kv_heads 1 .. 65535";
  if (c.block_size < kF8Span || c.block_size % kF8Span != 0)
    return "block_size must be a positive multiple of 16";
  if (static_cast<int64_t>(c.num_blocks) * (c.block_size / kF8Span) > INT32_MAX / c.num_kv_heads)
    return "num_blocks x block_size x num_kv_heads must be less than 2^35";
  return "";
}

std::string f8_cache_rows(const PthAttnCacheF8& c) {
  if (!c.k_cache.data || !c.v_cache.data || !c.k_scale || !c.v_scale)
    return "the cache's codes and scales must be non-NULL";
  for (const PthAttnStream* s : {&c.k_cache, &c.v_cache}) {
    const int64_t block = used_stride(s->stride_block, c.num_blocks);
    const int64_t head = used_stride(s->stride_head, c.num_kv_heads);
    if (reinterpret_cast<uintptr_t>(s->data) % 16 != 0 || block % 16 != 0 ||
        s->stride_slot % 16 != 0 || head % 16 != 0 || block < 0 || head < 0 ||
        s->stride_slot < 0 || s->stride_slot >= 1 << 24)
      return "k_cache and v_cache must have 16-byte aligned rows, strides >= 0 and less than 2^24 "
             "bytes between slots";
  }
  return "";
}

int32_t launch_write_f8(const PthAttnWriteF8Args& a, hipStream_t stream) {
  clear_error();
  PA_REQUIRE(a.abi_version == PTH_ATTN_ABI_VERSION,
             "abi_version " + std::to_string(a.abi_version) + " != library ABI " +
                 std::to_string(PTH_ATTN_ABI_VERSION));
  PA_REQUIRE(a.struct_bytes == static_cast<int32_t>(sizeof(PthAttnWriteF8Args)),
             "struct_bytes " + std::to_string(a.struct_bytes) + " != sizeof(PthAttnWriteF8Args) " +
                 std::to_string(sizeof(PthAttnWriteF8Args)));
  const std::string sizes = f8_cache_sizes(a.cache);
  PA_REQUIRE(sizes.empty(), sizes);
  PA_REQUIRE(a.kv_dtype == PTH_ATTN_F32 || a.kv_dtype == PTH_ATTN_F16 || a.kv_dtype == PTH_ATTN_BF16,
             "kv_dtype must be PTH_ATTN_F32, PTH_ATTN_F16 or PTH_ATTN_BF16");
  PA_REQUIRE(a.num_tokens >= 0 && a.num_tokens < 1 << 30, "num_tokens must be 0 .. 2^30 - 1");
  if (a.num_tokens == 0) return PTH_ATTN_OK;
  PA_REQUIRE(a.key && a.value && a.slot_mapping, "key, value and slot_mapping must be non-NULL");
  const std::string rows = f8_cache_rows(a.cache);
  PA_REQUIRE(rows.empty(), rows);
  const PthAttnCacheF8& c = a.cache;
  const int64_t elt = a.kv_dtype == PTH_ATTN_F32 ? 4 : 2;
  PA_REQUIRE(reinterpret_cast<uintptr_t>(a.key) % elt == 0 &&
                 reinterpret_cast<uintptr_t>(a.value) % elt == 0 &&
                 a.key_stride_token % elt == 0 && a.key_stride_head % elt == 0 &&
                 a.value_stride_token % elt == 0 && a.value_stride_head % elt == 0,
             "key and value must be aligned to their element");
  WriteF8Params w{};
  w.src[0] = static_cast<const char*>(a.key);
  w.src[1] = static_cast<const char*>(a.value);
  w.s_tok[0] = a.key_stride_token;
  w.s_tok[1] = a.value_stride_token;
  w.s_head[0] = a.key_stride_head;
  w.s_head[1] = a.value_stride_head;
  w.cache[0] = stream_of(c.k_cache);
  w.cache[1] = stream_of(c.v_cache);
  w.scale[0] = c.k_scale;
  w.scale[1] = c.v_scale;
  w.slot_mapping = a.slot_mapping;
  w.num_slots = static_cast<int64_t>(c.num_blocks) * c.block_size;
  w.n_sub = c.block_size / kF8Span;
  w.sub_div = Div32::make(static_cast<uint32_t>(w.n_sub));
  w.num_kv_heads = c.num_kv_heads;
  w.num_tokens = a.num_tokens;
  const int32_t cus = resident_workgroups();
  PA_REQUIRE(cus > 0, "cannot query the compute-unit count of the current device");
  w.tokens = 2;
  w.heads = 1;
  while (w.tokens <= 4 &&
         static_cast<int64_t>(a.num_tokens) * c.num_kv_heads > int64_t{4} * cus * w.tokens)
    w.tokens *= 2;
  const bool many = w.tokens > 4;
  if (many && a.num_tokens < kManyTokens) {
    w.tokens = 16;
    const int64_t units = static_cast<int64_t>((a.num_tokens + 15) / 16) * c.num_kv_heads;
    w.heads = static_cast<int32_t>((units + cus - 1) / cus);
  } else if (many) {
    const int64_t rounds = (int64_t{a.num_tokens} + kWriteTokens * cus - 1) / (kWriteTokens * cus);
    w.heads = c.num_kv_heads;
    w.tokens = static_cast<int32_t>((a.num_tokens + rounds * cus - 1) / (rounds * cus));
  }
  const bool wide = on16(a.key, a.key_stride_token, a.num_tokens, a.key_stride_head, c.num_kv_heads) &&
                    on16(a.value, a.value_stride_token, a.num_tokens, a.value_stride_head, c.num_kv_heads);
  const int64_t runs = (int64_t{a.num_tokens} + w.tokens - 1) / w.tokens;
  PA_REQUIRE(runs <= kMostThreads / (many ? kManyThreads : kThreads),
             "num_tokens needs more than 2^32 threads");
  const dim3 grid(static_cast<unsigned>(runs),
                  static_cast<unsigned>((c.num_kv_heads + w.heads - 1) / w.heads));
  switch (c.head_size) {
    case 64: write_d<64>(w, a.kv_dtype, wide, many, grid, stream); break;
    case 256: write_d<256>(w, a.kv_dtype, wide, many, grid, stream); break;
    default: write_d<128>(w, a.kv_dtype, wide, many, grid, stream);
  }
  const hipError_t err = hipGetLastError();
  if (err != hipSuccess)
    return fail(PTH_ATTN_ECUDA, std::string("8-bit cache writer launch: ") + hipGetErrorString(err));
  return PTH_ATTN_OK;
}

int32_t launch_gather_f8(const PthAttnGatherF8Args& a, hipStream_t stream) {
  clear_error();
  PA_REQUIRE(a.abi_version == PTH_ATTN_ABI_VERSION,
             "abi_version " + std::to_string(a.abi_version) + " != library ABI " +
                 std::to_string(PTH_ATTN_ABI_VERSION));
  PA_REQUIRE(a.struct_bytes == static_cast<int32_t>(sizeof(PthAttnGatherF8Args)),
             "struct_bytes " + std::to_string(a.struct_bytes) +
                 " != sizeof(PthAttnGatherF8Args) " + std::to_string(sizeof(PthAttnGatherF8Args)));
  const std::string sizes = f8_cache_sizes(a.cache);
  PA_REQUIRE(sizes.empty(), sizes);
  PA_REQUIRE(a.kv_dtype == PTH_ATTN_F32 || a.kv_dtype == PTH_ATTN_F16 || a.kv_dtype == PTH_ATTN_BF16,
             "kv_dtype must be PTH_ATTN_F32, PTH_ATTN_F16 or PTH_ATTN_BF16");
  PA_REQUIRE(a.num_tokens >= 0 && a.num_reqs >= 0 && a.num_reqs < 1 << 30 &&
                 a.block_table_width >= 0,
             "num_tokens and block_table_width must be >= 0, num_reqs 0 .. 2^30 - 1");
  if (a.num_tokens == 0 || a.num_reqs == 0) return PTH_ATTN_OK;
  PA_REQUIRE(a.key && a.value && a.row_start_loc, "key, value and row_start_loc must be non-NULL");
  PA_REQUIRE(a.block_table || a.block_table_width == 0, "block_table must be non-NULL");
  const std::string rows = f8_cache_rows(a.cache);
  PA_REQUIRE(rows.empty(), rows);
  const PthAttnCacheF8& c = a.cache;
  PA_REQUIRE(on16(a.key, a.key_stride_token, a.num_tokens, a.key_stride_head, c.num_kv_heads) &&
                 on16(a.value, a.value_stride_token, a.num_tokens, a.value_stride_head,
                      c.num_kv_heads),
             "key and value must have 16-byte aligned rows");
  GatherF8Params g{};
  g.dst[0] = static_cast<char*>(a.key);
  g.dst[1] = static_cast<char*>(a.value);
  g.s_tok[0] = a.key_stride_token;
  g.s_tok[1] = a.value_stride_token;
  g.s_head[0] = a.key_stride_head;
  g.s_head[1] = a.value_stride_head;
  g.cache[0] = stream_of(c.k_cache);
  g.cache[1] = stream_of(c.v_cache);
  g.scale[0] = c.k_scale;
  g.scale[1] = c.v_scale;
  g.block_table = a.block_table;
  g.bt_stride = a.block_table_row_stride;
  g.starts = a.row_start_loc;
  g.first = a.first;
  // A position is divided as 31 bits.
  g.reach = std::min<int64_t>(int64_t{a.block_table_width} * c.block_size, INT32_MAX);
  g.bs_div = Div32::make(static_cast<uint32_t>(c.block_size));
  g.n_sub = c.block_size / kF8Span;
  g.num_blocks = c.num_blocks;
  g.num_reqs = a.num_reqs;
  g.num_tokens = a.num_tokens;
  g.num_kv_heads = c.num_kv_heads;
  g.row_items = c.num_kv_heads * (c.head_size / (a.kv_dtype == PTH_ATTN_F32 ? 4 : 8));
  g.item_div = Div32::make(static_cast<uint32_t>(g.row_items));
  const int32_t cus = resident_workgroups();
  PA_REQUIRE(cus > 0, "cannot query the compute-unit count of the current device");
  // A work-group's rows: few enough for one turn of its threads; fewer where that leaves
  // compute units without a second work-group (8 heads of 128, 16, 8, 4 rows: 20,480
  // tokens 25.9, 24.0, 23.0 us, 1,024 7.8, 5.6, 4.4; one head, 20,480 5.6, 7.5, 8.8).
  g.tokens = kGatherTokens;
  while (g.tokens > 2 && (g.tokens * g.row_items > kPiecesAhead * kThreads / 2 ||
                          (g.tokens > 4 && a.num_tokens < 2 * cus * g.tokens)))
    g.tokens /= 2;
  const int64_t runs = (int64_t{a.num_tokens} + g.tokens - 1) / g.tokens;
  PA_REQUIRE(runs <= kMostThreads / kThreads, "num_tokens needs more than 2^32 threads");
  const dim3 grid(static_cast<unsigned>(runs));
  switch (c.head_size) {
    case 64: gather_d<64>(g, a.kv_dtype, grid, stream); break;
    case 256: gather_d<256>(g, a.kv_dtype, grid, stream); break;
    default: gather_d<128>(g, a.kv_dtype, grid, stream);
  }
  const hipError_t err = hipGetLastError();
  if (err != hipSuccess)
    return fail(PTH_ATTN_ECUDA, std::string("8-bit cache reader launch: ") + hipGetErrorString(err));
  return PTH_ATTN_OK;
}

}  // namespace pa

extern "C" {

int32_t pth_attn_write_f8_args_bytes(void) {
  return static_cast<int32_t>(sizeof(PthAttnWriteF8Args));
}
int32_t pth_attn_gather_f8_args_bytes(void) {
  return static_cast<int32_t>(sizeof(PthAttnGatherF8Args));
}

int32_t pth_attn_write_f8(const PthAttnWriteF8Args* args, void* stream) {
  if (args == nullptr) return pa::fail(PTH_ATTN_EINVAL, "args is NULL");
  return pa::launch_write_f8(*args, static_cast<hipStream_t>(stream));
}

int32_t pth_attn_gather_f8(const PthAttnGatherF8Args* args, void* stream) {
  if (args == nullptr) return pa::fail(PTH_ATTN_EINVAL, "args is NULL");
  return pa::launch_gather_f8(*args, static_cast<hipStream_t>(stream));
}

}  // extern "C"
