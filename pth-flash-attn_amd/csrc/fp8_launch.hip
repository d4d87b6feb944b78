// fp8_launch.hip -- host side of attention over a paged cache in 8-bit floating
// point: checks, the choice of kernel, the partition's size, and the C entry
// points.

#include <hip/hip_runtime.h>

#include <algorithm>
#include <climits>
#include <cmath>
#include <string>

#include "fp8.h"

namespace pa {
namespace {

// Slots per group up to which a larger team pays (p16_launch.hip has the measurements),
// and key rows that a work-group reads for each row of sums in its slots, below which the
// slots' bytes cost more than a larger team's reads save. One request, 8 heads of 128,
// teams of 1, 2, 4: 1,024 keys 10.3, 10.0, 11.0 us; 4,096 12.8, 12.1, 11.9; 131,072 66, 56,
// 52. 64 requests of 1,024 to 32,768 530, 447, 406.
constexpr int64_t kMostSlots = 128;
constexpr int64_t kLeastReads = 4;

bool rows_aligned(const void* p, int64_t a, int64_t b) {
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && a % 16 == 0 && b % 16 == 0;
}
CacheStream stream_of(const PthAttnStream& s) {
  return CacheStream{static_cast<const char*>(s.data), s.stride_block, s.stride_slot,
                     s.stride_head};
}

// Units that a work-group of the 16-row kernel computes side by side, one for
// each wave or pair of waves: neighbours in the cache (the KV heads of NHD
// pages), or row tiles of the same keys, as long as enough groups remain and,
// where they are cut, their slots stay small beside the keys. `rows`: a unit's.
int32_t team_of(const F8Params& p, int64_t span, int64_t rows, bool whole, int32_t cus) {
  const int64_t n_rt = p.qsl ? 1 : (p.group + kP16RowsRows - 1) / kP16RowsRows;
  const int64_t units = p.num_reqs * (p.num_kv_heads * n_rt);
  const bool heads_adjacent = p.k.s_head < p.k.s_slot && p.v.s_head < p.v.s_slot;
  const int64_t beside = heads_adjacent ? p.num_kv_heads * n_rt : n_rt;
  int32_t team = beside % 4 == 0 ? 4 : beside % 2 == 0 ? 2 : 1;
  while (team > 1 && units / team * kMostSlots < cus) team /= 2;
  while (!whole && team > 1 && units * span < kLeastReads * 2 * team * rows * cus) team /= 2;
  return team;
}

// The 16-row kernel's work-groups per compute unit where groups are cut: one of four
// units side by side (256 requests to 4,096 keys, 8 heads of 128, one and two 193 and 202
// us), more of fewer (1,024 requests to 1,000 keys, one head, one, two, three 59, 51, 63).
int64_t rows_per_cu(const F8Params& p, int32_t head_size, int64_t groups, int32_t cus) {
  if (p.team == 4) return 1;
  return std::min<int64_t>(p16_resident(head_size), std::max<int64_t>(1, groups / cus));
}

// Whether every group is left whole, so that there is nothing to join: where
// all are short. Decodes, whole and cut, 512 keys: 1 request and 1 KV head of 128
// 8.1 and 9.5 us, 64 and 8 heads 19.3 and 19.9; 768 keys 9.5 and 9.5, 26.4 and 25.2;
// 1,024 keys 12.3 and 10.0, 33.5 and 30.4. Heads of 64, 1,024 keys: 16 requests, 8 heads
// 10.3 and 11.2, 64 requests 25.5 and 22.8. Heads of 256, 64 requests, 4 heads, 256 keys
// 14.5 and 17.0, 512 keys 20.0 and 21.0, of one request 16.9 and 15.9.
bool whole_rows(int32_t head_size, int64_t span, int64_t units, int32_t cus) {
  if (head_size == 256) return span <= 256;
  return span <= (head_size == 64 && units <= cus / 2 ? 1024 : 512);
}

// The keys that a request of so many tokens may see: their last window + tokens - 1,
// from a block's beginning on.
int64_t span_of(const F8Params& p, int64_t tokens) {
  return p.window > 0 ? std::min<int64_t>(p.max_keys, int64_t{p.window} + tokens - 1 + 15)
                      : p.max_keys;
}

// Whether a batch whose longest request has `longest` tokens is one of prompts and
// decodes, so that requests of few rows get their own launch: eight of them, if the
// others are as long as the longest, and work enough for what that launch costs. Whole
// calls of decodes with prompts, 32 / 8 heads of 128, one launch and two: 60 of 2,000
// keys (123 MB) with 2 x 512 tokens 68 and 72 us, 90 122 and 94, 120 with 1 x 512 132 and
// 114, 200 of 1,000 with 2 x 32 140 and 116; 8 of 2,000 (21 MB) with 1 x 512 53 and 65, 20 of
// 1,000 with 4 x 8 29 and 46.
constexpr int64_t kMixedBytes = int64_t{1} << 27;  // of K, at the longest length
bool mixed(const F8Params& p, int32_t head_size, int64_t longest) {
  const int64_t few = p.num_reqs - (p.num_tokens + longest - 1) / longest;
  return p.group <= kP16RowsRows && few >= 8 &&
         few * span_of(p, 1) * p.num_kv_heads * head_size >= kMixedBytes;
}

// The kernel of few or many rows over the requests that p names, and the join.
// `longest`: of their query tokens (a choice only).
int32_t launch_part(F8Params p, int32_t head_size, bool f16, bool wide, int64_t longest,
                    int32_t cus, hipStream_t stream) {
  const int64_t bm = wide ? kP16WideRows : kP16RowsRows;
  // Bounds of the partition: row tiles and groups of all requests, key tiles of one.
  const int64_t rows = static_cast<int64_t>(p.num_tokens) * p.group;
  const int64_t reqs = p.num_reqs;
  int64_t row_tiles = rows / bm + reqs;
  if (p.qsl == nullptr) row_tiles = reqs * ((p.group + bm - 1) / bm);
  else if (p.most_rows <= bm) row_tiles = reqs;
  else if (p.least_rows > 0) row_tiles = rows / bm + std::min(reqs, rows / p.least_rows);
  int64_t tokens = p.qsl ? p.num_tokens : 1;
  if (p.qsl && p.most_rows <= bm) tokens = std::max<int64_t>(p.most_rows / p.group, 1);
  const int64_t span = span_of(p, tokens);
  const int64_t units = row_tiles * p.num_kv_heads;
  if (units == 0) return PTH_ATTN_OK;
  const bool whole = wide ? f8_whole_wide(head_size, span, units, cus)
                          : whole_rows(head_size, span, units, cus);
  p.team = wide ? 1 : team_of(p, span, std::min(bm, longest * p.group), whole, cus);
  // Fewer units side by side while compute units lack work-groups, and further only
  // where all of a unit's waves have keys (8 heads of 128, 128 keys, one unit and two: 16
  // requests 6.9 and 7.5 us, 64 requests 8.8 and 8.0).
  if (whole)
    while (p.team > 1 && (units / p.team < cus ||
                          (units / p.team < p16_resident(head_size) * cus &&
                           64 * 2 * kP16Waves / p.team <= span + 63)))
      p.team /= 2;
  // 64-key tiles of many rows are shared out by what a unit sees (f8_steps), so that a
  // group left whole has larger ones.
  p.key_tile_log2 = wide ? (whole ? 7 : 6) : 8 - (p.team >> 1);
  if (whole)
    while ((int64_t{1} << p.key_tile_log2) < span) ++p.key_tile_log2;
  p.slot_rows = static_cast<int32_t>(p.qsl ? bm : std::min<int64_t>(bm, p.group));
  const int64_t key_tiles =
      std::max<int64_t>((span + (1 << p.key_tile_log2) - 1) >> p.key_tile_log2, 1);
  const int64_t groups =
      p.qsl == nullptr ? reqs * ((row_tiles / reqs * p.num_kv_heads + p.team - 1) / p.team)
                       : units / p.team + (p.team > 1 ? reqs : 0);
  // The shares of causal units are up to six tiles each more than their keys (F8Steps).
  PA_REQUIRE(units < INT32_MAX / (key_tiles + 6), "the launch exceeds 2^31 tiles");
  const int64_t fill =
      cus * (wide ? p16_resident(head_size) : rows_per_cu(p, head_size, groups, cus));
  p.num_wg = static_cast<int32_t>(std::min(groups * key_tiles, fill));
  const bool cuts = wide ? !whole : key_tiles > 1;
  if (!cuts)
    p.num_wg = static_cast<int32_t>(std::min<int64_t>(groups, (wide ? 64 : 8) * cus));
  p.notes = !cuts ? -1 : groups <= p.num_wg ? static_cast<int32_t>(groups) : 0;
  hipError_t err = wide ? launch_f8_wide_kernel(p, f16, head_size, stream)
                        : launch_f8_rows_kernel(p, f16, head_size, stream);
  // Work-groups of the join per note (p16_launch.hip has the measurements).
  const int32_t items = p.team * p.slot_rows, least = wide ? 16 : 1;
  const int32_t y =
      p.notes > 0 ? std::min(items, std::max(least, (wide ? 8 : 4) * cus / p.notes)) : least;
  if (err == hipSuccess && cuts)
    err = launch_f8_combine_kernel(p, f16, wide, head_size, y, stream);
  if (err != hipSuccess)
    return fail(PTH_ATTN_ECUDA,
                std::string("paged 8-bit attention launch: ") + hipGetErrorString(err));
  return PTH_ATTN_OK;
}

}  // namespace

int32_t launch_paged_f8(const PthAttnPagedF8Args& a, hipStream_t stream) {
  clear_error();
  PA_REQUIRE(a.abi_version == PTH_ATTN_ABI_VERSION,
             "abi_version " + std::to_string(a.abi_version) + " != library ABI " +
                 std::to_string(PTH_ATTN_ABI_VERSION));
  PA_REQUIRE(a.struct_bytes == static_cast<int32_t>(sizeof(PthAttnPagedF8Args)),
             "struct_bytes " + std::to_string(a.struct_bytes) + " != sizeof(PthAttnPagedF8Args) " +
                 std::to_string(sizeof(PthAttnPagedF8Args)));
  const PthAttnCacheF8& c = a.cache;
  const std::string sizes = f8_cache_sizes(c);
  PA_REQUIRE(sizes.empty(), sizes);
  PA_REQUIRE(a.dtype == PTH_ATTN_F16 || a.dtype == PTH_ATTN_BF16,
             "dtype must be PTH_ATTN_F16 or PTH_ATTN_BF16");
  PA_REQUIRE(a.num_reqs >= 0 && a.num_tokens >= 0, "num_reqs and num_tokens must be >= 0");
  PA_REQUIRE(a.num_q_heads >= 1 && a.num_q_heads % c.num_kv_heads == 0,
             "num_q_heads must be a positive multiple of num_kv_heads");
  PA_REQUIRE(a.num_q_heads / c.num_kv_heads <= 64, "at most 64 query heads per KV head");
  PA_REQUIRE(a.query_start_loc != nullptr || a.num_tokens == a.num_reqs,
             "without query_start_loc, num_tokens must equal num_reqs");
  PA_REQUIRE(a.window >= 0, "window must be >= 0");
  PA_REQUIRE(a.window == 0 || a.causal, "a window needs causal");
  PA_REQUIRE(a.max_kv_len >= 0 && a.block_table_width >= 0,
             "max_kv_len and block_table_width must be >= 0");
  PA_REQUIRE(std::isfinite(a.softmax_scale) && a.softmax_scale > 0.0f,
             "softmax_scale must be finite and > 0");
  if (a.num_reqs == 0 || a.num_tokens == 0) return PTH_ATTN_OK;
  PA_REQUIRE(a.q && a.out && a.kv_lens, "q, out and kv_lens must be non-NULL");
  PA_REQUIRE(a.block_table || a.block_table_width == 0, "block_table must be non-NULL");
  PA_REQUIRE(rows_aligned(a.q, used_stride(a.q_stride_token, a.num_tokens),
                          used_stride(a.q_stride_head, a.num_q_heads)) &&
                 rows_aligned(a.out, used_stride(a.out_stride_token, a.num_tokens),
                              used_stride(a.out_stride_head, a.num_q_heads)),
             "q and out must have 16-byte aligned rows");
  const std::string bad = f8_cache_rows(c);
  PA_REQUIRE(bad.empty(), bad);
  const int32_t cus = resident_workgroups();
  PA_REQUIRE(cus > 0, "cannot query the compute-unit count of the current device");
  const int64_t need = p16_workspace_floats(c.head_size, cus);
  PA_REQUIRE(a.ws && reinterpret_cast<uintptr_t>(a.ws) % 16 == 0 && a.ws_floats >= need,
             "ws must be 16-byte aligned and hold " + std::to_string(need) + " floats, holds " +
                 std::to_string(a.ws_floats));

  F8Params p{};
  p.q = static_cast<const char*>(a.q);
  p.s_q_tok = a.q_stride_token;
  p.s_q_head = a.q_stride_head;
  p.out = static_cast<char*>(a.out);
  p.s_out_tok = a.out_stride_token;
  p.s_out_head = a.out_stride_head;
  p.k = stream_of(c.k_cache);
  p.v = stream_of(c.v_cache);
  p.block_table = a.block_table;
  p.bt_stride = a.block_table_row_stride;
  p.kv_lens = a.kv_lens;
  p.qsl = a.query_start_loc;
  p.ws = a.ws;
  p.group = a.num_q_heads / c.num_kv_heads;
  p.bs_div = Div32::make(static_cast<uint32_t>(c.block_size));
  p.g_div = Div32::make(static_cast<uint32_t>(p.group));
  p.num_blocks = c.num_blocks;
  const int64_t reach = static_cast<int64_t>(a.block_table_width) * c.block_size;
  p.max_keys = static_cast<int32_t>(
      std::min({static_cast<int64_t>(a.max_kv_len), reach, int64_t{kF8MostKeys}}));
  p.num_reqs = a.num_reqs;
  p.num_tokens = a.num_tokens;
  p.num_kv_heads = c.num_kv_heads;
  p.window = a.window < p.max_keys ? a.window : 0;
  p.scale_log2 = a.softmax_scale * 1.4426950408889634f;
  p.k_exp = c.k_scale;
  p.v_exp = c.v_scale;
  p.n_sub = c.block_size / kF8Span;
  p.causal = a.causal ? 1 : 0;

  const int64_t rows = static_cast<int64_t>(a.num_tokens) * p.group;
  PA_REQUIRE(rows < INT32_MAX - 1024, "num_tokens x heads per KV head exceeds 2^31");
  p.least_rows = 0;
  p.most_rows = INT32_MAX;
  const int64_t longest = a.query_start_loc ? std::max(a.max_query_len, 1) : 1;
  const bool wide = longest * p.group > kP16RowsRows && a.query_start_loc != nullptr;
  if (!wide || !mixed(p, c.head_size, longest))
    return launch_part(p, c.head_size, a.dtype == PTH_ATTN_F16, wide,
                       std::max<int64_t>(longest, 1), cus, stream);
  // Requests of up to 16 rows by one kernel, the others by the other.
  F8Params few = p;
  p.least_rows = kP16RowsRows + 1;
  few.most_rows = kP16RowsRows;
  const int32_t rc =
      launch_part(p, c.head_size, a.dtype == PTH_ATTN_F16, true, longest, cus, stream);
  if (rc != PTH_ATTN_OK) return rc;
  return launch_part(few, c.head_size, a.dtype == PTH_ATTN_F16, false,
                     std::max<int64_t>(kP16RowsRows / p.group, 1), cus, stream);
}

}  // namespace pa

extern "C" {

int32_t pth_attn_paged_f8_args_bytes(void) { return static_cast<int32_t>(sizeof(PthAttnPagedF8Args)); }

int64_t pth_attn_paged_f8_workspace_floats(int32_t head_size) {
  return pth_attn_paged16_workspace_floats(head_size);
}

int32_t pth_attn_paged_f8(const PthAttnPagedF8Args* args, void* stream) {
  if (args == nullptr) return pa::fail(PTH_ATTN_EINVAL, "args is NULL");
  return pa::launch_paged_f8(*args, static_cast<hipStream_t>(stream));
}

}  // extern "C"
