// p16_launch.hip -- host side of attention over a paged 16-bit cache: checks,
// the choice of kernel, the partition's size, and the C entry points.

#include <hip/hip_runtime.h>

#include <algorithm>
#include <climits>
#include <cmath>
#include <string>

#include "p16.h"

namespace pa {
namespace {

// Slots per group up to which a larger team pays (one request to 128k keys, 32q /
// 8kv of 128: 96.6, 86.8 and 83.6 us for teams of 1, 2 and 4, which has 128; the
// join takes 4.6 to 4.8).
constexpr int64_t kMostSlots = 128;
// Key rows that a work-group reads for each row of sums in its slots, below
// which the slots' bytes cost more than a larger team's reads save. Whole call,
// teams of 1, 2 and 4 (with 4: the ratio), 4 tokens per request, 32q / 8kv of 128:
//     8 requests to 1,500 states (2.9)  18.1, 18.1, 20.1 us
//    16                          (5.9)  27.0, 25.6, 27.0
//     8             6,000       (11.7)  43.3, 40.5, 41.0
//     2            30,000       (14.6)  53.4, 49.2, 48.5
constexpr int64_t kLeastReads = 8;

// A stride of a dimension of n elements, as far as it is used.
int64_t used(int64_t stride, int64_t n) { return n > 1 ? stride : 0; }
bool rows_aligned(const void* p, int64_t a, int64_t b) {
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && a % 16 == 0 && b % 16 == 0;
}
bool stream_ok(const PthAttnStream& s, const PthAttnP16Args& a) {
  const int64_t block = used(s.stride_block, a.num_blocks);
  const int64_t slot = used(s.stride_slot, a.block_size);
  const int64_t head = used(s.stride_head, a.num_kv_heads);
  return rows_aligned(s.data, block, slot) && head % 16 == 0 && block >= 0 && head >= 0 &&
         slot >= 0 && slot < (1 << 24);
}
CacheStream stream_of(const PthAttnStream& s) {
  return CacheStream{static_cast<const char*>(s.data), s.stride_block, s.stride_slot,
                     s.stride_head};
}

// Units that a work-group of the 16-row kernel computes side by side, one for
// each wave or pair of waves: neighbours in the cache (the KV heads of NHD
// pages), or row tiles of the same keys, as long as enough groups remain and,
// where they are cut, their slots stay small beside the keys. `rows`: a unit's.
int32_t team_of(const P16Params& p, int64_t span, int64_t rows, bool whole, int32_t cus) {
  const int64_t n_rt = p.qsl ? 1 : (p.group + kP16RowsRows - 1) / kP16RowsRows;
  const int64_t units = p.num_reqs * (p.num_kv_heads * n_rt);
  const bool heads_adjacent = p.k.s_head < p.k.s_slot && p.v.s_head < p.v.s_slot;
  const int64_t beside = heads_adjacent ? p.num_kv_heads * n_rt : n_rt;
  int32_t team = beside % 4 == 0 ? 4 : beside % 2 == 0 ? 2 : 1;
  while (team > 1 && units / team * kMostSlots < cus) team /= 2;
  while (!whole && team > 1 && units * span < kLeastReads * 2 * team * rows * cus) team /= 2;
  return team;
}

// The 16-row kernel's work-groups per compute unit where groups are cut. One,
// four waves, reads the cache fastest: more streams at once cost the memory more
// than they hide (64 requests to 32k keys at D = 128: 626 us with one, 646 with
// two, 652 with three). Where a work-group takes several groups, others fill the
// gaps between them, as many as fit (48 requests to 4k, 16 heads of 64 in HND
// pages: 92 us with one, 78 with two, 76 with three).
int64_t rows_per_cu(int32_t head_size, int64_t groups, int32_t cus) {
  return std::min<int64_t>(p16_resident(head_size), std::max<int64_t>(1, groups / cus));
}

// Whether every group is left whole, so that there is nothing to join: where
// all are short. Measured, whole call, cut and whole, 32q / 8kv of 128, requests
// of one token (bounds of 64, 256, 512 and 1,024 keys):
//     8 requests  10.7, 6.5   11.5,  8.6   12.6, 12.0   15.1, 20.5 us
//    64           11.9, 7.5   19.3, 14.8   25.7, 24.6   40.0, 44.2
// D = 64 is alike; at D = 256, with one work-group per compute unit, 8 requests
// of one token take 12.7, 9.7 and 13.3, 14.4 at 64 and 256.
bool whole_rows(int32_t head_size, int64_t span) {
  return span <= (head_size == 256 ? 128 : 512);
}
// The same of 128-row units, whose slots are larger and so joined later: requests
// of 25 to 100 tokens against a third of so many states or more (700, 1,000,
// 1,500, 2,000), 32q / 8kv of 128:
//     1 request   17.2, 17.1   16.0, 20.9   17.4, 27.2
//     6 requests  28.8, 21.8   30.0, 28.6   33.8, 37.9   35.6, 48.6
//    20           46.1, 30.0   52.8, 36.5   62.0, 54.0   71.8, 69.3
//    28           56.5, 49.1   67.0, 66.7   81.6, 90.8   99.6, 115
//    64          107.2, 84.3  130.5, 108   169.1, 148
// 20 requests' units all but fill the device once, and then longer ones may stay
// whole, too (D = 64 likewise: 53.3, 44.2 at 1,500); many units of one request,
// whose lengths are alike, cost the end of the last (8 requests of 4,000 tokens:
// 238, 239 at 500 and 341, 391 at 1,000; 16 of 2,000 255, 225 and 355, 358). At
// D = 256, 16q / 4kv: 8 requests 38.6, 34.0 at 500, 43.5, 54.9 at 1,000; 16, three
// quarters of the device, 58.0, 52.7; 400, whose shares are many short units,
// 418, 445 at 500. The bounds are bands of the units' number, not costs, and miss
// two lines above: 64 requests at 1,500 (three rounds of units) and 20 at 2,000 are
// cut.
bool whole_wide(int32_t head_size, int64_t span, int64_t units, int32_t cus) {
  const int64_t round = int64_t{p16_resident(head_size)} * cus;
  int64_t most = head_size == 256 ? 512 : 1024;
  if (units < cus / 8 || units > 8 * cus) most = head_size == 256 ? 128 : 512;
  else if (10 * units >= 7 * round && units <= round) most = 1536;
  return span <= most;
}

}  // namespace

int32_t launch_p16(const PthAttnP16Args& a, hipStream_t stream) {
  clear_error();
  PA_REQUIRE(a.abi_version == PTH_ATTN_ABI_VERSION,
             "abi_version " + std::to_string(a.abi_version) + " != library ABI " +
                 std::to_string(PTH_ATTN_ABI_VERSION));
  PA_REQUIRE(a.struct_bytes == static_cast<int32_t>(sizeof(PthAttnP16Args)),
             "struct_bytes " + std::to_string(a.struct_bytes) + " != sizeof(PthAttnP16Args) " +
                 std::to_string(sizeof(PthAttnP16Args)));
  PA_REQUIRE(a.head_size == 64 || a.head_size == 128 || a.head_size == 256,
             "head_size must be 64, 128 or 256");
  PA_REQUIRE(a.dtype == PTH_ATTN_F16 || a.dtype == PTH_ATTN_BF16,
             "dtype must be PTH_ATTN_F16 or PTH_ATTN_BF16");
  PA_REQUIRE(a.num_reqs >= 0 && a.num_tokens >= 0 && a.num_blocks >= 1 && a.block_size >= 1,
             "num_reqs, num_tokens >= 0, num_blocks and block_size >= 1");
  PA_REQUIRE(a.num_kv_heads >= 1 && a.num_q_heads >= 1 && a.num_q_heads % a.num_kv_heads == 0,
             "num_q_heads must be a positive multiple of num_kv_heads");
  PA_REQUIRE(a.num_q_heads / a.num_kv_heads <= 64, "at most 64 query heads per KV head");
  PA_REQUIRE(a.query_start_loc != nullptr || a.num_tokens == a.num_reqs,
             "without query_start_loc, num_tokens must equal num_reqs");
  PA_REQUIRE(a.query_start_loc == nullptr || a.window == 0,
             "a window needs one query token per request");
  PA_REQUIRE(a.window >= 0, "window must be >= 0");
  PA_REQUIRE(a.max_kv_len >= 0 && a.block_table_width >= 0,
             "max_kv_len and block_table_width must be >= 0");
  PA_REQUIRE(std::isfinite(a.softmax_scale) && a.softmax_scale > 0.0f,
             "softmax_scale must be finite and > 0");
  if (a.num_reqs == 0 || a.num_tokens == 0) return PTH_ATTN_OK;
  PA_REQUIRE(a.q && a.out && a.k_cache.data && a.v_cache.data && a.kv_lens,
             "q, out, k_cache, v_cache and kv_lens must be non-NULL");
  PA_REQUIRE(a.block_table || a.block_table_width == 0, "block_table must be non-NULL");
  PA_REQUIRE(rows_aligned(a.q, used(a.q_stride_token, a.num_tokens),
                          used(a.q_stride_head, a.num_q_heads)) &&
                 rows_aligned(a.out, used(a.out_stride_token, a.num_tokens),
                              used(a.out_stride_head, a.num_q_heads)),
             "q and out must have 16-byte aligned rows");
  PA_REQUIRE(stream_ok(a.k_cache, a) && stream_ok(a.v_cache, a),
             "k_cache and v_cache must have 16-byte aligned rows, strides >= 0 and less than "
             "2^24 bytes between slots");
  const int32_t cus = resident_workgroups();
  PA_REQUIRE(cus > 0, "cannot query the compute-unit count of the current device");
  const int64_t need = p16_workspace_floats(a.head_size, cus);
  PA_REQUIRE(a.ws && reinterpret_cast<uintptr_t>(a.ws) % 16 == 0 && a.ws_floats >= need,
             "ws must be 16-byte aligned and hold " + std::to_string(need) + " floats, holds " +
                 std::to_string(a.ws_floats));

  P16Params p{};
  p.q = static_cast<const char*>(a.q);
  p.s_q_tok = a.q_stride_token;
  p.s_q_head = a.q_stride_head;
  p.out = static_cast<char*>(a.out);
  p.s_out_tok = a.out_stride_token;
  p.s_out_head = a.out_stride_head;
  p.k = stream_of(a.k_cache);
  p.v = stream_of(a.v_cache);
  p.block_table = a.block_table;
  p.bt_stride = a.block_table_row_stride;
  p.kv_lens = a.kv_lens;
  p.qsl = a.query_start_loc;
  p.ws = a.ws;
  p.group = a.num_q_heads / a.num_kv_heads;
  p.bs_div = Div32::make(static_cast<uint32_t>(a.block_size));
  p.g_div = Div32::make(static_cast<uint32_t>(p.group));
  p.num_blocks = a.num_blocks;
  const int64_t reach = static_cast<int64_t>(a.block_table_width) * a.block_size;
  // Key positions stay below 2^31 with a tile to spare.
  const int64_t most = INT32_MAX - 1024;
  p.max_keys = static_cast<int32_t>(std::min({static_cast<int64_t>(a.max_kv_len), reach, most}));
  p.num_reqs = a.num_reqs;
  p.num_tokens = a.num_tokens;
  p.num_kv_heads = a.num_kv_heads;
  p.window = a.window;
  p.scale_log2 = a.softmax_scale * 1.4426950408889634f;

  // More rows than the small kernel's tile of a KV head: the other, whose tiles
  // eight times as many rows share. Whole call, small kernel and wide one, 1, 8
  // and 64 requests against 1,500 states:
  //                    16 rows                             20 rows
  //   16q / 16kv of 64 13.0, 13.9  18.0, 17.4  76.4, 82.1  11.8, 14.3  25.7, 16.9  117, 83.4 us
  //   32q / 8kv of 128 13.0, 12.2  18.5, 18.3  75.1, 78.0  13.5, 12.3  27.3, 18.6  105, 78.3
  //   16q / 4kv of 256 16.5, 16.6  22.5, 22.8  76.8, 85.7  17.4, 17.0  28.3, 23.1  119, 86.0
  // One request at D = 64 would keep the small one.
  const bool wide = a.query_start_loc != nullptr &&
                    static_cast<int64_t>(a.max_query_len) * p.group > kP16RowsRows;
  const int64_t bm = wide ? kP16WideRows : kP16RowsRows;
  const int64_t rows = static_cast<int64_t>(a.num_tokens) * p.group;
  PA_REQUIRE(rows < INT32_MAX - 1024, "num_tokens x heads per KV head exceeds 2^31");
  // Bounds of the partition: groups of all requests, key tiles of one.
  const int64_t row_tiles = a.query_start_loc == nullptr
                                ? a.num_reqs * ((p.group + bm - 1) / bm)
                                : rows / bm + a.num_reqs;
  const int64_t span = p.window > 0 ? std::min<int64_t>(p.max_keys, int64_t{p.window} + 15)
                                    : p.max_keys;
  const int64_t units = row_tiles * a.num_kv_heads;
  const bool whole =
      wide ? whole_wide(a.head_size, span, units, cus) : whole_rows(a.head_size, span);
  const int64_t tokens = a.query_start_loc ? std::max(a.max_query_len, 1) : 1;
  p.team = wide ? 1 : team_of(p, span, std::min(bm, tokens * p.group), whole, cus);
  if (whole)
    while (p.team > 1 && units / p.team < p16_resident(a.head_size) * cus) p.team /= 2;
  p.key_tile_log2 = wide ? 6 : 7 - (p.team >> 1);
  if (whole)
    while ((int64_t{1} << p.key_tile_log2) < span) ++p.key_tile_log2;
  p.slot_rows = static_cast<int32_t>(a.query_start_loc ? bm : std::min<int64_t>(bm, p.group));
  const int64_t key_tiles =
      std::max<int64_t>((span + (1 << p.key_tile_log2) - 1) >> p.key_tile_log2, 1);
  const int64_t groups =
      a.query_start_loc == nullptr
          ? a.num_reqs * ((row_tiles / a.num_reqs * a.num_kv_heads + p.team - 1) / p.team)
          : units / p.team + (p.team > 1 ? a.num_reqs : 0);
  PA_REQUIRE(units < INT32_MAX / key_tiles, "the launch exceeds 2^31 tiles");
  const int64_t fill =
      cus * (wide ? p16_resident(a.head_size) : rows_per_cu(a.head_size, groups, cus));
  p.num_wg = static_cast<int32_t>(std::min(groups * key_tiles, fill));
  if (key_tiles == 1) p.num_wg = static_cast<int32_t>(std::min<int64_t>(groups, 8 * cus));
  p.notes = key_tiles == 1 ? -1 : groups <= p.num_wg ? static_cast<int32_t>(groups) : 0;
  const bool f16 = a.dtype == PTH_ATTN_F16, page16 = a.block_size % 16 == 0;
  hipError_t err = wide ? launch_p16_wide_kernel(p, f16, page16, a.head_size, stream)
                        : launch_p16_rows_kernel(p, f16, page16, a.head_size, stream);
  // Work-groups of the join per note: a row or eight each, until the device is
  // full (256 tokens against 4,096 states: 23 us with one, 8.3 with eight).
  // Of 16-row units, four times as many as compute units (4 tokens of 8 requests
  // against 1,500 states, D = 256: whole call 29.1 us with twice, 25.7). Of 128-row
  // units at least 16, a row of a work-group's crew each (28 requests of 25 to 100
  // tokens to 2,000 states 88.9 us with 4, 86.4; others alike within 1 %).
  const int32_t items = p.team * p.slot_rows, least = wide ? 16 : 1;
  const int32_t y =
      p.notes > 0 ? std::min(items, std::max(least, (wide ? 8 : 4) * cus / p.notes)) : least;
  if (err == hipSuccess && key_tiles > 1)
    err = launch_p16_combine_kernel(p, f16, wide, a.head_size, y, stream);
  if (err != hipSuccess)
    return fail(PTH_ATTN_ECUDA, std::string("paged16 launch: ") + hipGetErrorString(err));
  return PTH_ATTN_OK;
}

}  // namespace pa

extern "C" {

int32_t pth_attn_paged16_args_bytes(void) { return static_cast<int32_t>(sizeof(PthAttnP16Args)); }

int64_t pth_attn_paged16_workspace_floats(int32_t head_size) {
  const int32_t cus = pa::resident_workgroups();
  return cus > 0 ? pa::p16_workspace_floats(head_size, cus) : 0;
}

int32_t pth_attn_paged16(const PthAttnP16Args* args, void* stream) {
  if (args == nullptr) return pa::fail(PTH_ATTN_EINVAL, "args is NULL");
  return pa::launch_p16(*args, static_cast<hipStream_t>(stream));
}

}  // extern "C"
