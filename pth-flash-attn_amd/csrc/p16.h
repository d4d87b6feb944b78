// p16.h -- attention over a paged cache in the model's own 16-bit type:
// launch parameters, and the partition of the work that its kernels share
// (p16_rows.hip: units of 16 query rows; p16_wide.hip: units of 128;
// p16_combine.hip: joins what the partition cut).
//
// The work of a launch is a stream of key tiles. A unit is a row tile (kRows
// consecutive rows, a row being a (query token, query head of the KV head)
// pair) of one request and one KV head; it has ceil(keys / kKeys) tiles, one
// if it sees no key. Units lie end to end, requests first, then KV heads,
// then row tiles. Work-group w of W takes tiles [w N / W, (w + 1) N / W) of
// the N (W at most N, so that none between two of a unit's is without tiles):
// equal shares whatever the lengths, and at most two units of a work-group are
// cut, its first and its last. A cut unit leaves unnormalised
// partial sums in the workspace, two slots per work-group whatever the batch:
// slot 2 w for a range that begins inside a unit, 2 w + 1 for one that begins
// with it. The combine's work-group w joins the unit whose beginning w holds.
//
// Everything is a function of the device's lengths and of launch constants,
// so a captured graph replays as the lengths change.

#pragma once

#include "attn_stream.h"

namespace pa {

struct P16Params {
  const char* q;
  int64_t s_q_tok, s_q_head;
  char* out;
  int64_t s_out_tok, s_out_head;
  CacheStream k, v;
  const int32_t* block_table;
  int64_t bt_stride;  // elements
  const int32_t* kv_lens;
  const int32_t* qsl;  // nullptr: request r has the one query token r
  float* ws;
  Div32 bs_div;  // slots per page
  Div32 g_div;   // query heads per KV head
  int32_t num_blocks;
  int32_t max_keys;  // no request has more (the table's reach and the caller's bound)
  int32_t num_reqs;
  int32_t num_tokens;
  int32_t num_kv_heads;
  int32_t group;
  int32_t window;
  int32_t num_wg;
  float scale_log2;  // softmax_scale * log2(e)
};

// Key tile and row tile of the two kernels.
constexpr int kP16Waves = 4;
constexpr int kP16RowsRows = 16, kP16RowsKeys = 32 * kP16Waves;
constexpr int kP16WideRows = 32 * kP16Waves, kP16WideKeys = 64;

// Floats of workspace per compute unit: the most that a kernel's resident
// work-groups need, two slots of kRows * (D + 2) each.
constexpr int kP16WsRowsPerCu = 512;
inline int64_t p16_workspace_floats(int32_t head_size, int32_t cus) {
  return static_cast<int64_t>(cus) * kP16WsRowsPerCu * (head_size + 2);
}

#if defined(__HIPCC__)

// A request as the partition sees it. Starts and lengths outside their
// tensors' range are brought into it: the kernels read and write nothing
// outside whatever the lengths say.
struct P16Req {
  int32_t q0;    // first query token
  int32_t rows;  // query tokens x group
  int32_t lo;    // first visible key
  int32_t base;  // lo rounded down to a 16-key block
  int32_t len;   // one past the last
  int32_t n_rt;  // row tiles
  int32_t n_kt;  // key tiles, >= 1
};

template <int kRows, int kKeys>
__device__ __forceinline__ P16Req p16_request_of(const P16Params& p, int r, int q0, int q1,
                                                 int len) {
  P16Req x;
  if (p.qsl == nullptr) {
    q0 = r;
    q1 = r + 1;
  }
  x.q0 = min(max(q0, 0), p.num_tokens);
  x.rows = max(min(q1, p.num_tokens) - x.q0, 0) * p.group;
  x.len = min(max(len, 0), p.max_keys);
  x.lo = p.window > 0 ? max(x.len - p.window, 0) : 0;
  x.base = x.lo & ~15;
  x.n_rt = (x.rows + kRows - 1) / kRows;
  x.n_kt = max((x.len - x.base + kKeys - 1) / kKeys, 1);
  return x;
}

template <int kRows, int kKeys>
__device__ __forceinline__ int64_t p16_tiles(const P16Params& p, const P16Req& x) {
  return static_cast<int64_t>(p.num_kv_heads) * x.n_rt * x.n_kt;
}

// Tiles of request `r` by vector loads (r differs from lane to lane).
template <int kRows, int kKeys>
__device__ __forceinline__ int64_t p16_lane_tiles(const P16Params& p, int r) {
  if (r >= p.num_reqs) return 0;
  int len = p.kv_lens[r], q0 = 0, q1 = 0;
  if (p.qsl != nullptr) {
    q0 = p.qsl[r];
    q1 = p.qsl[r + 1];
  }
  return p16_tiles<kRows, kKeys>(p, p16_request_of<kRows, kKeys>(p, r, q0, q1, len));
}

// Forward-only walk over the requests, 64 at a time (every lane the same but
// for `incl`).
struct P16Cursor {
  int r0;
  int64_t base, end;  // tiles before request r0, and through r0 + 63
  int64_t incl;       // the lane's inclusive prefix within the 64
};

// All tiles of the launch; the cursor at its first 64 requests.
template <int kRows, int kKeys>
__device__ __forceinline__ int64_t p16_begin(const P16Params& p, P16Cursor& c, int lane) {
  c.r0 = 0;
  c.base = 0;
  c.incl = wave_scan64(p16_lane_tiles<kRows, kKeys>(p, lane), lane);
  c.end = readlane64(c.incl, 63);
  int64_t more = 0;
  for (int r0 = 64; r0 < p.num_reqs; r0 += 64) more += p16_lane_tiles<kRows, kKeys>(p, r0 + lane);
  if (p.num_reqs <= 64) return c.end;
  return c.end + readlane64(wave_scan64(more, lane), 63);
}

// A unit, and the tile of it that a position falls on.
struct P16Unit {
  P16Req req;
  int32_t r, head, rt, kt;
};

// The unit of tile `at` (not before the cursor, and less than all tiles).
template <int kRows, int kKeys>
__device__ __forceinline__ P16Unit p16_locate(const P16Params& p, P16Cursor& c, int64_t at,
                                              int lane) {
  while (at >= c.end && c.r0 + 64 < p.num_reqs) {
    c.r0 += 64;
    c.base = c.end;
    c.incl = wave_scan64(p16_lane_tiles<kRows, kKeys>(p, c.r0 + lane), lane);
    c.end = c.base + readlane64(c.incl, 63);
  }
  const int64_t local = at - c.base;
  const int j = min(static_cast<int>(__popcll(__ballot(c.incl <= local))), 63);
  const int64_t before = j > 0 ? readlane64(c.incl, j - 1) : 0;
  P16Unit u;
  u.r = __builtin_amdgcn_readfirstlane(min(c.r0 + j, p.num_reqs - 1));
  int len = ld_ro(p.kv_lens, u.r), q0 = 0, q1 = 0;
  if (p.qsl != nullptr) {
    q0 = ld_ro(p.qsl, u.r);
    q1 = ld_ro(p.qsl, u.r + 1);
  }
  u.req = p16_request_of<kRows, kKeys>(p, u.r, q0, q1, len);
  // Within a request: less than 2^31 tiles, by the launcher's check.
  const uint32_t in_req = static_cast<uint32_t>(local - before);
  const uint32_t unit = in_req / static_cast<uint32_t>(u.req.n_kt);
  u.kt = static_cast<int32_t>(in_req - unit * static_cast<uint32_t>(u.req.n_kt));
  const uint32_t n_rt = static_cast<uint32_t>(max(u.req.n_rt, 1));
  u.head = static_cast<int32_t>(unit / n_rt);
  u.rt = static_cast<int32_t>(unit - static_cast<uint32_t>(u.head) * n_rt);
  u.r = __builtin_amdgcn_readfirstlane(u.r);
  u.head = __builtin_amdgcn_readfirstlane(u.head);
  u.rt = __builtin_amdgcn_readfirstlane(u.rt);
  u.kt = __builtin_amdgcn_readfirstlane(u.kt);
  return u;
}

// Work-groups that take tiles.
__device__ __forceinline__ int p16_takers(const P16Params& p, int64_t tiles) {
  return static_cast<int>(min(tiles, static_cast<int64_t>(p.num_wg)));
}
// The first tile of work-group w (w at most num_wg, num_wg > 0).
__device__ __forceinline__ int64_t p16_share(int64_t tiles, int w, int num_wg) {
  return tiles * w / num_wg;
}
// The work-group that holds tile `at`.
__device__ __forceinline__ int p16_holder(int64_t tiles, int64_t at, int num_wg) {
  return static_cast<int>(((at + 1) * num_wg + tiles - 1) / tiles) - 1;
}

// Slot `i`'s partial sums and its (maximum, sum) pairs.
template <int kRows, int D>
__device__ __forceinline__ float* p16_slot_o(const P16Params& p, int i) {
  return p.ws + static_cast<int64_t>(i) * kRows * D;
}
template <int kRows, int D>
__device__ __forceinline__ float* p16_slot_ml(const P16Params& p, int i) {
  return p.ws + static_cast<int64_t>(2) * p.num_wg * kRows * D + static_cast<int64_t>(i) * kRows * 2;
}

// The address of row `row` (within its unit's row tile): query token and head.
template <int kRows>
__device__ __forceinline__ void p16_row(const P16Params& p, const P16Unit& u, int row,
                                        int64_t& token, int64_t& head) {
  const uint32_t i = static_cast<uint32_t>(u.rt * kRows + row);
  const uint32_t t = p.g_div.div(i);
  token = u.req.q0 + static_cast<int64_t>(t);
  head = static_cast<int64_t>(u.head) * p.group + (i - t * static_cast<uint32_t>(p.group));
}

#endif  // __HIPCC__

// Host side.
int32_t launch_p16(const PthAttnP16Args& a, hipStream_t stream);
hipError_t launch_p16_rows_kernel(const P16Params& p, bool f16, bool page16, int head_size,
                                  hipStream_t stream);
hipError_t launch_p16_wide_kernel(const P16Params& p, bool f16, bool page16, int head_size,
                                  hipStream_t stream);
hipError_t launch_p16_combine_kernel(const P16Params& p, bool f16, bool wide, int head_size,
                                     hipStream_t stream);
int32_t launch_write_kv16(const PthAttnWrite16Args& a, hipStream_t stream);
int32_t launch_step_tables(const PthAttnTablesArgs& a, hipStream_t stream);

}  // namespace pa
