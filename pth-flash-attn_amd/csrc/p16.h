// p16.h -- attention over a paged cache in the model's own 16-bit type:
// launch parameters, and the partition of the work that its kernels share
// (p16_rows.hip: units of 16 query rows; p16_wide.hip: units of 128;
// p16_combine.hip: joins what the partition cut).
//
// The work of a launch is a stream of key tiles. A unit is a row tile (kRows
// consecutive rows, a row being a (query token, query head of the KV head)
// pair) of one request and one KV head; units lie requests first, then KV
// heads, then row tiles. A group is `team` consecutive units of a request that
// a work-group computes side by side; it has ceil(keys / key_tile) tiles, one
// if it sees no key. Groups lie end to end, and work-group w of W takes tiles
// [w N / W, (w + 1) N / W) of the N (W at most N, so that none between two of a
// group's is without tiles): equal shares whatever the lengths, and at most
// two groups of a work-group are cut, its first and its last. A cut group
// leaves unnormalised partial sums in the workspace, two slots per work-group
// whatever the batch: slot 2 w for a range that begins inside a group, 2 w + 1
// for one that begins with it. The work-group that holds a group's beginning
// notes how it was cut (P16Cut), for the combine, which joins it. The note's
// place is the group's number where the launch has few groups, so that the
// combine needs no work-groups for nothing, and the work-group's otherwise.
//
// Everything is a function of the device's lengths and of launch constants,
// so a captured graph replays as the lengths change.

#pragma once

#include "attn_stream.h"
#include "p16_geometry.h"

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
  int32_t team;           // units of a group: 1, 2 or 4
  int32_t key_tile_log2;  // keys of a tile
  int32_t slot_rows;      // rows of a unit that a slot holds: no unit has more
  // Notes by group number: at most so many; 0: by work-group; -1: none, no
  // group is cut.
  int32_t notes;
  float scale_log2;       // softmax_scale * log2(e)
};

// A cut group: the slots that hold it (0: none is cut) and, above kP16CutShift,
// the work-group that begins it; its request's first query token and rows, its
// place among the request's groups.
struct P16Cut {
  uint32_t slots_wg;
  int32_t q0, rows, group;
};
constexpr int kP16CutShift = 16;

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
  int32_t n_gr;  // groups of units
  int32_t n_kt;  // key tiles, >= 1
};

template <int kRows>
__device__ __forceinline__ P16Req p16_request_of(const P16Params& p, int r, int q0, int q1,
                                                 int len) {
  P16Req x;
  if (p.qsl == nullptr) {
    q0 = r;
    q1 = r + 1;
  }
  const P16Tokens t = p16_tokens(q0, q1, p.num_tokens);
  x.q0 = t.first;
  x.rows = t.count * p.group;
  x.len = min(max(len, 0), p.max_keys);
  x.lo = p.window > 0 ? max(x.len - p.window, 0) : 0;
  x.base = x.lo & ~15;
  x.n_rt = (x.rows + kRows - 1) / kRows;
  x.n_gr = (p.num_kv_heads * x.n_rt + p.team - 1) >> (p.team >> 1);  // / team
  x.n_kt = max((x.len - x.base + (1 << p.key_tile_log2) - 1) >> p.key_tile_log2, 1);
  return x;
}

// Length and first and last query token of request `r` (r differs from lane to
// lane; none behind the last request).
struct P16Lane {
  int32_t len, q0, q1;
};
__device__ __forceinline__ P16Lane p16_lane(const P16Params& p, int r) {
  P16Lane x = {0, 0, 0};
  if (r < p.num_reqs) {
    x.len = p.kv_lens[r];
    if (p.qsl != nullptr) {
      x.q0 = p.qsl[r];
      x.q1 = p.qsl[r + 1];
    }
  }
  return x;
}
// Its tiles and groups.
struct P16Count {
  int64_t tiles;
  int32_t groups;
};
template <int kRows>
__device__ __forceinline__ P16Count p16_count(const P16Params& p, const P16Lane& n, int r) {
  if (r >= p.num_reqs) return {0, 0};
  const P16Req x = p16_request_of<kRows>(p, r, n.q0, n.q1, n.len);
  return {static_cast<int64_t>(x.n_gr) * x.n_kt, x.n_gr};
}

// Walk over the requests, 64 (a window) at a time. Lane i knows its request of
// the window, and, up to 64 windows, how many tiles and groups end with window
// i, so that a work-group goes to its own at once.
struct P16Cursor {
  int r0;             // the window's first request
  int64_t base, end;  // tiles before it, and through it
  int64_t incl;       // the lane's inclusive prefix within it
  int32_t groups, group_incl;  // groups before it; the lane's prefix (p16_counted)
  P16Lane of;                  // the lane's request
  int64_t window_end;
  int32_t window_groups;
};

// Groups are counted beside the tiles where their number is the note's place
// and the requests have different ones.
__device__ __forceinline__ bool p16_counted(const P16Params& p) {
  return p.notes > 0 && p.qsl != nullptr;
}

// The cursor at the 64 requests from r0 on.
template <int kRows>
__device__ __forceinline__ void p16_window(const P16Params& p, P16Cursor& c, int lane) {
  c.of = p16_lane(p, c.r0 + lane);
  const P16Count n = p16_count<kRows>(p, c.of, c.r0 + lane);
  c.incl = wave_scan64(n.tiles, lane);
  c.end = c.base + readlane64(c.incl, 63);
  if (p16_counted(p)) c.group_incl = wave_scan32(n.groups);
}

// All tiles of the launch; the cursor at its first window.
template <int kRows>
__device__ __forceinline__ int64_t p16_begin(const P16Params& p, P16Cursor& c, int lane) {
  c.r0 = 0;
  c.base = 0;
  c.groups = 0;
  c.group_incl = 0;
  p16_window<kRows>(p, c, lane);
  if (p.num_reqs <= 64) return c.end;
  int64_t all = c.end;
  int32_t groups = p16_counted(p) ? __builtin_amdgcn_readlane(c.group_incl, 63) : 0;
  c.window_end = all;
  c.window_groups = groups;
#pragma unroll 2
  for (int w = 1; w < (p.num_reqs + 63) >> 6; ++w) {
    const int r = 64 * w + lane;
    const P16Count n = p16_count<kRows>(p, p16_lane(p, r), r);
    all += readlane64(wave_scan64(n.tiles, lane), 63);
    if (p16_counted(p)) groups += __builtin_amdgcn_readlane(wave_scan32(n.groups), 63);
    if (lane >= w) {
      c.window_end = all;
      c.window_groups = groups;
    }
  }
  return all;
}

// A group, and the tile of it that a position falls on.
struct P16Group {
  P16Req req;
  int32_t r, group, kt;
  int32_t number;  // of the request's first group, where it counts (p16_counted)
};

// The group of tile `at` (not before the cursor, and less than all tiles).
template <int kRows>
__device__ __forceinline__ P16Group p16_locate(const P16Params& p, P16Cursor& c, int64_t at,
                                               int lane) {
  if (at >= c.end && p.num_reqs > 64) {
    // Past the 64th window, which says what all after it hold, one by one.
    const int w = static_cast<int>(__popcll(__ballot(c.window_end <= at)));
    if (c.r0 < 64 * 63 && w > 0) {
      const int to = min(w, 63);
      c.r0 = 64 * to;
      c.base = readlane64(c.window_end, to - 1);
      c.groups = __builtin_amdgcn_readlane(c.window_groups, to - 1);
      p16_window<kRows>(p, c, lane);
    }
    while (at >= c.end && c.r0 + 64 < p.num_reqs) {
      c.r0 += 64;
      c.base = c.end;
      c.groups += __builtin_amdgcn_readlane(c.group_incl, 63);
      p16_window<kRows>(p, c, lane);
    }
  }
  const int64_t local = at - c.base;
  const int j = __builtin_amdgcn_readfirstlane(
      min(static_cast<int>(__popcll(__ballot(c.incl <= local))), 63));
  const int64_t before = j > 0 ? readlane64(c.incl, j - 1) : 0;
  P16Group u;
  u.number = c.groups + (j > 0 ? __builtin_amdgcn_readlane(c.group_incl, j - 1) : 0);
  u.r = __builtin_amdgcn_readfirstlane(min(c.r0 + j, p.num_reqs - 1));
  u.req = p16_request_of<kRows>(p, u.r, __builtin_amdgcn_readlane(c.of.q0, j),
                                __builtin_amdgcn_readlane(c.of.q1, j),
                                __builtin_amdgcn_readlane(c.of.len, j));
  // Within a request: less than 2^31 tiles, by the launcher's check.
  const uint32_t in_req = static_cast<uint32_t>(local - before);
  const uint32_t n_kt = static_cast<uint32_t>(u.req.n_kt);
  u.group = __builtin_amdgcn_readfirstlane(static_cast<int32_t>(in_req / n_kt));
  u.kt = __builtin_amdgcn_readfirstlane(static_cast<int32_t>(in_req)) -
         u.group * static_cast<int32_t>(n_kt);
  return u;
}

// Work-groups that take tiles.
__device__ __forceinline__ int p16_takers(const P16Params& p, int64_t tiles) {
  return static_cast<int>(min(tiles, static_cast<int64_t>(p.num_wg)));
}
// The first tile of work-group w (w at most num_wg, num_wg > 0).
__device__ __forceinline__ int64_t p16_share(int64_t tiles, int w, int num_wg) {
  const uint64_t x = static_cast<uint64_t>(tiles) * static_cast<uint32_t>(w);
  if (x >> 32 == 0) return static_cast<uint32_t>(x) / static_cast<uint32_t>(num_wg);
  return static_cast<int64_t>(x / static_cast<uint32_t>(num_wg));
}
// The work-group that holds tile `at`.
__device__ __forceinline__ int p16_holder(int64_t tiles, int64_t at, int num_wg) {
  const uint64_t x = static_cast<uint64_t>(at + 1) * static_cast<uint32_t>(num_wg) +
                     static_cast<uint64_t>(tiles) - 1;
  if (x >> 32 == 0)
    return static_cast<int>(static_cast<uint32_t>(x) / static_cast<uint32_t>(tiles)) - 1;
  return static_cast<int>(x / static_cast<uint64_t>(tiles)) - 1;
}

// A unit: KV head and row tile.
struct P16Unit {
  int32_t head, rt;
};
__device__ __forceinline__ P16Unit p16_unit(const P16Req& x, int32_t index) {
  const uint32_t n = static_cast<uint32_t>(max(x.n_rt, 1));
  P16Unit u;
  u.head = n == 1 ? index : static_cast<int32_t>(static_cast<uint32_t>(index) / n);
  u.rt = n == 1 ? 0 : index - u.head * static_cast<int32_t>(n);
  return u;
}

// Row `row` of a slot's unit `sub`: D sums, and their maximum and weight sum.
// A slot holds slot_rows rows of each unit: one long request's many slots are
// read together, and lie as close as they can.
template <int D>
__device__ __forceinline__ float* p16_slot_o(const P16Params& p, int slot, int sub, int row) {
  return p.ws + (static_cast<int64_t>(slot * p.team + sub) * p.slot_rows + row) * D;
}
template <int D>
__device__ __forceinline__ float* p16_slot_ml(const P16Params& p, int slot, int sub, int row) {
  const int64_t rows = static_cast<int64_t>(2) * p.num_wg * p.team * p.slot_rows;
  return p.ws + rows * D + (static_cast<int64_t>(slot * p.team + sub) * p.slot_rows + row) * 2;
}
template <int D>
__device__ __forceinline__ P16Cut* p16_cut(const P16Params& p, int i) {
  return reinterpret_cast<P16Cut*>(p16_slot_ml<D>(p, 2 * p.num_wg, 0, 0)) + i;
}
// Notes that work-group wg begins the group `gr`, cut or (`cut` false) whole.
template <int D>
__device__ __forceinline__ void p16_note(const P16Params& p, const P16Group& gr, int wg,
                                         int64_t tiles, int64_t first, int takers, bool cut) {
  P16Cut c = {0u, gr.req.q0, gr.req.rows, gr.group};
  if (cut) {
    const int last = p16_holder(tiles, first + gr.req.n_kt - 1, takers);
    c.slots_wg = static_cast<uint32_t>(last - wg + 1) | static_cast<uint32_t>(wg) << kP16CutShift;
  }
  // Starts that run backwards can make more groups than there are notes.
  const int number = (p16_counted(p) ? gr.number : gr.r * gr.req.n_gr) + gr.group;
  if (p.notes == 0 || static_cast<uint32_t>(number) < static_cast<uint32_t>(p.notes))
    *p16_cut<D>(p, p.notes ? 1 + number : wg) = c;
}
template <int D>
__device__ __forceinline__ void p16_note_none(const P16Params& p, int wg) {
  if (p.notes == 0) p16_cut<D>(p, wg)->slots_wg = 0u;
}
// The note before the first group's: how many groups there are. By the first
// work-group, in any case.
template <int kRows, int D>
__device__ __forceinline__ void p16_note_groups(const P16Params& p, const P16Cursor& c, int lane) {
  if (!p16_counted(p)) return;
  int32_t n = __builtin_amdgcn_readlane(c.group_incl, 63);
  for (int r0 = 64; r0 < p.num_reqs; r0 += 64)
    n += __builtin_amdgcn_readlane(
        wave_scan32(p16_count<kRows>(p, p16_lane(p, r0 + lane), r0 + lane).groups), 63);
  if (threadIdx.x == 0) p16_cut<D>(p, 0)->slots_wg = static_cast<uint32_t>(n);
}

// Query token and head of row `row` of a unit.
template <int kRows>
__device__ __forceinline__ void p16_row(const P16Params& p, int32_t q0, const P16Unit& u, int row,
                                        int64_t& token, int64_t& head) {
  const uint32_t i = static_cast<uint32_t>(u.rt * kRows + row);
  const uint32_t t = p.g_div.div(i);
  token = q0 + static_cast<int64_t>(t);
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
                                     int y, hipStream_t stream);
int32_t launch_write_kv16(const PthAttnWrite16Args& a, hipStream_t stream);
int32_t launch_step_tables(const PthAttnTablesArgs& a, hipStream_t stream);

}  // namespace pa
