// step_tables.hip -- a step's block tables and slot map from its request
// lengths (pth_attn_step_tables in include/pth_attn.h has the formulas).
//
// Two prefix sums over the requests, of the new tokens and of the pages that
// they need, and then independent look-ups: the page of a new token is in the
// request's row if it existed before, in the free list otherwise, so nothing
// waits for what another work-group writes. Each work-group therefore makes the
// prefix sums itself, a chunk of requests at a time in LDS, and takes of each
// chunk its own new tokens (binary search for the request), its share of the
// pages and of the requests' own outputs: one launch, no atomics in memory.
// Sums saturate at kCap, above every bound that they are compared with.
//
// Bound: latency, of the launch and two dependent reads (lengths, page), with the
// steps of a search in LDS between them: 8 requests of one token 3.2 us, 1,024
// requests with 33,000 new tokens 7.3 us.

#include <hip/hip_runtime.h>

#include <algorithm>
#include <string>

#include "attn_stream.h"
#include "p16.h"

namespace pa {
namespace {

constexpr uint32_t kCap = 1u << 30;
// New tokens per work-group: one per thread, whose search and read are one
// chain. 1,024 requests with 33,000 new tokens: 9.9 us with four per thread.
constexpr int kTokens = 256;

struct TablesParams {
  int32_t* block_table;
  int64_t bt_stride;
  int64_t* slot_mapping;
  int32_t* seq_lens;
  int32_t* query_start_loc;
  int32_t* pool_out;
  const int32_t* context_lens;
  const int32_t* query_lens;
  const int32_t* free_pages;
  const int32_t* pool_in;
  uint32_t num_free, num_slots;
  int32_t width, num_reqs;
  Div32 bs_div;
};

__device__ __forceinline__ uint32_t add_cap(uint32_t a, uint32_t b) {
  return min(a + b, kCap);  // both <= kCap
}

// Inclusive saturating prefix sum over the wave (wave_scan32's lane moves).
template <int kCtrl, int kRowMask = 0xf>
__device__ __forceinline__ uint32_t add_moved(uint32_t x) {
  return add_cap(x, static_cast<uint32_t>(dpp_i32<kCtrl, kRowMask>(static_cast<int>(x))));
}
__device__ __forceinline__ uint32_t wave_scan_cap(uint32_t x) {
  x = add_moved<0x111>(x);
  x = add_moved<0x112>(x);
  x = add_moved<0x114>(x);
  x = add_moved<0x118>(x);
  x = add_moved<0x142, 0xa>(x);
  return add_moved<0x143, 0xc>(x);
}

template <int kItems>
__global__ __launch_bounds__(256) void step_tables(const TablesParams p) {
  constexpr int kChunk = 256 * kItems;
  // Of the chunk's requests: tokens through it, its context, pages through it
  // (counted from the first of the step), and where its pages begin in the
  // free list, or kRefused.
  __shared__ uint32_t s_end[kChunk], s_ctx[kChunk], s_page[kChunk], s_first[kChunk];
  __shared__ uint32_t s_tok[4], s_new[4];
  __shared__ uint32_t s_taken, s_refused;
  constexpr uint32_t kRefused = 0xffffffffu;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const uint32_t bs = p.bs_div.d;
  const uint32_t reach = static_cast<uint32_t>(p.width) * bs;  // < 2^31
  const uint32_t cursor0 = static_cast<uint32_t>(max(p.pool_in[0], 0));
  const uint32_t cursor = min(cursor0, kCap);
  const uint32_t t0 = blockIdx.x * static_cast<uint32_t>(kTokens);
  const uint32_t t1 = min(t0 + kTokens, p.num_slots);
  if (tid == 0) {
    s_taken = 0;
    s_refused = 0;
  }
  uint32_t tokens = 0, pages = 0;  // of the chunks before
  for (int r0 = 0, chunk = 0; r0 < p.num_reqs; r0 += kChunk, ++chunk) {
    uint32_t ctx[kItems], n[kItems], add[kItems], tok_sum = 0, new_sum = 0;
    bool wide[kItems];
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
      const int r = r0 + kItems * tid + i;
      const bool in = r < p.num_reqs;
      ctx[i] = in ? static_cast<uint32_t>(max(p.context_lens[r], 0)) : 0u;
      n[i] = in ? static_cast<uint32_t>(max(p.query_lens[r], 0)) : 0u;
    }
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
      const uint32_t all = ctx[i] + n[i];
      wide[i] = all <= reach;
      const uint32_t have = p.bs_div.div(min(ctx[i], reach) + bs - 1);
      const uint32_t need = p.bs_div.div(min(all, reach) + bs - 1);
      add[i] = wide[i] ? min(need - have, kCap) : 0u;
      tok_sum = add_cap(tok_sum, min(n[i], kCap));
      new_sum = add_cap(new_sum, add[i]);
    }
    const uint32_t tok_incl = wave_scan_cap(tok_sum), new_incl = wave_scan_cap(new_sum);
    if (lane == 63) {
      s_tok[wave] = tok_incl;
      s_new[wave] = new_incl;
    }
    __syncthreads();
    uint32_t tok_at = tokens, new_at = pages;  // before this thread's requests
#pragma unroll
    for (int v = 0; v < 3; ++v) {
      tok_at = v < wave ? add_cap(tok_at, s_tok[v]) : tok_at;
      new_at = v < wave ? add_cap(new_at, s_new[v]) : new_at;
    }
    const uint32_t tok_up = __shfl_up(tok_incl, 1), new_up = __shfl_up(new_incl, 1);
    if (lane > 0) {
      tok_at = add_cap(tok_at, tok_up);
      new_at = add_cap(new_at, new_up);
    }
    const bool mine = chunk % static_cast<int>(gridDim.x) == static_cast<int>(blockIdx.x);
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
      const int r = r0 + kItems * tid + i;
      const uint32_t first = add_cap(cursor, new_at);
      const bool fits = wide[i] && (add[i] == 0 || first + add[i] <= p.num_free);
      if (r < p.num_reqs && mine) {
        p.seq_lens[r] = static_cast<int32_t>(fits ? ctx[i] + n[i] : ctx[i]);
        p.query_start_loc[r] = static_cast<int32_t>(min(tok_at, p.num_slots));
      }
      if (r < p.num_reqs && blockIdx.x == 0) {
        if (!fits) atomicAdd(&s_refused, 1u);
        else if (add[i] != 0) atomicMax(&s_taken, new_at + add[i]);
      }
      tok_at = add_cap(tok_at, min(n[i], kCap));
      new_at = add_cap(new_at, add[i]);
      const int at = kItems * tid + i;
      s_end[at] = tok_at;
      s_ctx[at] = ctx[i];
      s_page[at] = new_at;
      s_first[at] = fits ? first : kRefused;
      if (r == p.num_reqs - 1 && mine)
        p.query_start_loc[p.num_reqs] = static_cast<int32_t>(min(tok_at, p.num_slots));
    }
    __syncthreads();
    const int count = min(kChunk, p.num_reqs - r0);
    const uint32_t tok_end = s_end[count - 1], page_end = s_page[count - 1];
    // The first request of the chunk whose running sum passes x.
    auto find = [&](const uint32_t* sums, uint32_t x) {
      int lo = 0;
#pragma unroll
      for (int step = kChunk / 2; step > 0; step >>= 1)
        if (lo + step <= count - 1 && sums[lo + step - 1] <= x) lo += step;
      return lo;
    };
    // This work-group's new tokens among the chunk's.
    for (uint32_t t = max(t0, tokens) + tid; t < min(t1, tok_end); t += 256) {
      const int i = find(s_end, t);
      const uint32_t before = i > 0 ? s_end[i - 1] : tokens;
      const uint32_t c = s_ctx[i], pos = c + (t - before), first = s_first[i];
      int64_t slot = -1;
      if (first != kRefused) {
        const uint32_t j = p.bs_div.div(pos), have = p.bs_div.div(c + bs - 1);
        const int32_t page = j < have
                                 ? p.block_table[static_cast<int64_t>(r0 + i) * p.bt_stride + j]
                                 : p.free_pages[first + (j - have)];
        if (page >= 0) slot = static_cast<int64_t>(page) * bs + (pos - j * bs);
      }
      p.slot_mapping[t] = slot;
    }
    // Its share of the chunk's new pages, those that the free list holds.
    const uint32_t held = min(page_end, p.num_free - min(cursor, p.num_free));
    for (uint32_t x = pages + 256u * blockIdx.x + tid; x < held; x += 256u * gridDim.x) {
      const int i = find(s_page, x);
      const uint32_t before = i > 0 ? s_page[i - 1] : pages;
      const uint32_t first = s_first[i], k = x - before;
      if (first == kRefused) continue;
      const uint32_t have = p.bs_div.div(s_ctx[i] + bs - 1);
      p.block_table[static_cast<int64_t>(r0 + i) * p.bt_stride + have + k] =
          p.free_pages[first + k];
    }
    tokens = tok_end;
    pages = page_end;
    __syncthreads();
  }
  for (uint32_t t = max(t0, tokens) + tid; t < t1; t += 256) p.slot_mapping[t] = -1;
  if (blockIdx.x == 0 && tid == 0) {
    if (p.num_reqs == 0) p.query_start_loc[0] = 0;
    p.pool_out[0] = static_cast<int32_t>(cursor0 + s_taken);
    p.pool_out[1] = static_cast<int32_t>(s_refused);
  }
}

}  // namespace

int32_t launch_step_tables(const PthAttnTablesArgs& a, hipStream_t stream) {
  clear_error();
  PA_REQUIRE(a.abi_version == PTH_ATTN_ABI_VERSION,
             "abi_version " + std::to_string(a.abi_version) + " != library ABI " +
                 std::to_string(PTH_ATTN_ABI_VERSION));
  PA_REQUIRE(a.struct_bytes == static_cast<int32_t>(sizeof(PthAttnTablesArgs)),
             "struct_bytes " + std::to_string(a.struct_bytes) + " != sizeof(PthAttnTablesArgs) " +
                 std::to_string(sizeof(PthAttnTablesArgs)));
  PA_REQUIRE(a.num_reqs >= 0 && a.num_slots >= 0 && a.num_free >= 0 && a.block_table_width >= 0 &&
                 a.block_size >= 1,
             "num_reqs, num_slots, num_free and block_table_width >= 0, block_size >= 1");
  PA_REQUIRE(a.num_reqs < (1 << 30) && a.num_slots < kCap && a.num_free < kCap,
             "num_reqs, num_slots and num_free must be less than 2^30");
  PA_REQUIRE(static_cast<int64_t>(a.block_table_width) * a.block_size + a.block_size < 0x7fffffff,
             "block_table_width x block_size must be less than 2^31");
  PA_REQUIRE(a.query_start_loc && a.pool_out && a.pool_in,
             "query_start_loc, pool_out and pool_in must be non-NULL");
  PA_REQUIRE(a.num_reqs == 0 || (a.seq_lens && a.context_lens && a.query_lens),
             "seq_lens, context_lens and query_lens must be non-NULL");
  PA_REQUIRE(a.num_slots == 0 || a.slot_mapping, "slot_mapping must be non-NULL");
  PA_REQUIRE(a.num_reqs == 0 || a.block_table_width == 0 || a.block_table,
             "block_table must be non-NULL");
  PA_REQUIRE(a.num_reqs <= 1 || a.block_table_row_stride >= a.block_table_width,
             "the rows of block_table must not overlap");
  PA_REQUIRE(a.num_free == 0 || a.free_pages, "free_pages must be non-NULL");
  TablesParams p{};
  p.block_table = a.block_table;
  p.bt_stride = a.block_table_row_stride;
  p.slot_mapping = a.slot_mapping;
  p.seq_lens = a.seq_lens;
  p.query_start_loc = a.query_start_loc;
  p.pool_out = a.pool_out;
  p.context_lens = a.context_lens;
  p.query_lens = a.query_lens;
  p.free_pages = a.free_pages;
  p.pool_in = a.pool_in;
  p.num_free = static_cast<uint32_t>(a.num_free);
  p.num_slots = static_cast<uint32_t>(a.num_slots);
  p.width = a.block_table_width;
  p.num_reqs = a.num_reqs;
  p.bs_div = Div32::make(static_cast<uint32_t>(a.block_size));
  const int64_t work_groups = (a.num_slots + kTokens - 1) / kTokens;
  const dim3 grid(static_cast<unsigned>(std::max<int64_t>(work_groups, 1))), block(256);
  if (a.num_reqs <= 256) hipLaunchKernelGGL(step_tables<1>, grid, block, 0, stream, p);
  else hipLaunchKernelGGL(step_tables<4>, grid, block, 0, stream, p);
  const hipError_t err = hipGetLastError();
  if (err != hipSuccess)
    return fail(PTH_ATTN_ECUDA, std::string("step tables launch: ") + hipGetErrorString(err));
  return PTH_ATTN_OK;
}

}  // namespace pa

extern "C" {

int32_t pth_attn_tables_args_bytes(void) { return static_cast<int32_t>(sizeof(PthAttnTablesArgs)); }

int32_t pth_attn_step_tables(const PthAttnTablesArgs* args, void* stream) {
  if (args == nullptr) return pa::fail(PTH_ATTN_EINVAL, "args is NULL");
  return pa::launch_step_tables(*args, static_cast<hipStream_t>(stream));
}

}  // extern "C"
