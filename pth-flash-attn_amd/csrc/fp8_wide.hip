// fp8_wide.hip -- attention of many query rows over a paged cache in 8-bit
// floating point (fp8.h): prompts and long drafts, causal or not. A unit is 128
// rows of one KV head (p16.h), 32 for each of four waves, which share the key
// tiles of 64 in LDS.
//
// Layout. As p16_wide.hip: v_mfma_f32_32x32x16 with the keys (or the output
// columns) on M and the wave's query rows on N, K and V row-major in LDS, V read
// by columns with ds_read_b64_tr_b16. The codes come through registers: a wave
// loads the 16 keys of one block of scales, a tile ahead, converts them once for
// all four waves (two values an instruction, the scale with them) and stores
// them as 16-bit values. Conversion at the products would be done four times,
// and products of codes would take the queries and the weights apart into codes.
//
// Numerics. Scores, m, l and o are 32 bits; the running maximum moves only when
// a score passes it by 2^kSlack, so most tiles rescale nothing; P is scaled by
// 2^-kBias, so that sums of values near the type's largest do not leave 32
// bits. bf16: K's and V's values are exact, P is rounded once, to 8 bits, and l sums
// the rounded P: as in the 16-bit cache's kernel that is an error of the output's own
// size and independent of it (against 64 bits 0.0022 of an output's size, with an exact P
// 0.0017), and the rest of P would be a second PV product (fp16, below: 760 us for 533).
// fp16: K's codes are exact in fp16, their scale is a factor of the
// scores; V is in bf16, whose range its values need, and P a bf16 pair hi + lo.
// A row does not see the keys behind its own, nor the slots behind the request's
// last key in their block: where one of these has a NaN in V, it is taken out of the
// products of the tile and put back into the rows that do see it.
//
// Bound: the SIMDs' issue. 4 requests of 2,048 rows against 4,096 keys, 32 heads over 8
// of 128, 533 us, 1,031 TFLOP/s: matrix instructions 47 % of the cycles, vector ones
// (softmax, conversions) 50 %. The two can go on at once: a product of 32 cycles with four
// additions behind it takes 34, of one wave, and of two waves of a SIMD one's products
// keep their rate beside the other's additions, these 83 % of theirs. In batches they do
// so less (sixteen products, then 64 additions: 51 cycles a product, 40 with two waves),
// and a tile is batches, of scores, softmax and PV, that a barrier starts together in
// all waves. So codes are converted once for four waves, and nothing else is asked of a
// tile than its softmax needs. Heads of 64 339 us. Heads of 256, 16 over 8, 709 us:
// registers for one wave of a SIMD alone, and 64 KB written to LDS and 256 KB read for a
// tile, at some 80 bytes a cycle.

#include "fp8_device.h"

namespace pa {
namespace {

template <int D>
struct WideOf {
  static constexpr int kPerSimd = p16_resident(D);  // a work-group has a wave on each SIMD
  static constexpr int kQ = D / 16;       // QK products per 32 keys
  static constexpr int kO = D / 32;       // output tiles
  static constexpr int kRow = 2 * D;      // bytes of a key row in LDS
  static constexpr int kCodes = D / 16;   // 16-code pieces of a row in the cache
  static constexpr int kBuf = kP16WideKeys * kRow;
  static constexpr int kLoads = D / 64;   // loads of a wave per tile and stream
  // Units left whole of more keys than 2^(kSort - 1) go by length, others request by
  // request. Ragged batches gain, even ones of short units lose: 5 prompts of 500 to 2,500
  // tokens behind 100 to 6,200 keys, 8 heads of 128, 323 and 388 us, 16 of 1,024 232 and 221,
  // 16 of 256 49 and 39; 4 heads of 256, 4 of 1,024 81 and 104, 16 of 512 113 and 132.
  static constexpr int kSort = D == 256 ? 9 : 10;
  // Whether the next tile's addresses are asked for before the scores (heads of 256, one
  // wave on a SIMD: 716 and 709 us; heads of 128 533 and 540), or where they are needed.
  static constexpr bool kEarly = D == 256;
  // The place of 16-byte piece c of row t in LDS. Stores of 8 lanes, every second
  // piece of a row, take all 32 banks, reads (the same piece of 16 rows of K, four
  // of 4 rows of V) all 64.
  static __device__ __forceinline__ int k_piece(int t, int c) {
    if constexpr (D == 64) return c ^ (t & 1) ^ ((t >> 1) & 7);
    return (((c >> 1) & 7) ^ (t & 7)) | ((c ^ (t >> 3)) & 1) << 3 | (c >> 4) << 4;
  }
  static __device__ __forceinline__ int v_piece(int t, int c) {
    if constexpr (D == 64) return ((c >> 1) ^ (t & 2)) | ((c ^ t) & 1) << 2;
    return (((c >> 1) & 7) ^ 2 * (t & 3)) | ((c ^ t) & 1) << 3 | (c >> 4) << 4;
  }
  // A piece and the next, apart.
  static constexpr uint32_t kOddK = D == 64 ? 16 : 128, kOddV = D == 64 ? 64 : 128;
  // In K, a row and the i-th after it that a lane stores, apart.
  static __device__ __forceinline__ uint32_t k_row(int i) {
    return D == 128 ? 128u * i : 64u * (i & 1) | 128u * (i >> 1);
  }
};

// Units that are left whole by the keys that they see, most first, so that all
// compute units end together: unit `at` of that order, of up to 64 requests (a lane knows
// its own). A causal request's row tile rt sees prefix + 128 (rt + 1) / G keys or its
// window, so that it has a count of units with more than x keys in closed form, and a
// search over x (in steps of 64 keys, at most 128) finds the step that holds the unit.
// Within a step requests follow each other, and KV heads in turn: eight of them an XCD
// each, whose L2 has their keys.
__device__ __forceinline__ P16Group f8_longest(const F8Params& p, const P16Cursor& c, int32_t at,
                                               int lane, P16Unit& u) {
  const P16Req x = p16_request_of<kP16WideRows>(p, lane, c.of.q0, c.of.q1, c.of.len);
  const int n_rt = lane < p.num_reqs ? x.n_rt : 0;
  const bool grows = p.causal && p.qsl != nullptr;
  const int per = 128 / p.group + 1;  // tokens of a unit
  const int cap = p.window > 0 ? p.window + per : INT32_MAX;
  const int prefix =
      grows ? x.len - static_cast<int>(p.g_div.div(static_cast<uint32_t>(x.rows))) : x.len;
  const int most = __builtin_amdgcn_readfirstlane(
      wave_max32(n_rt > 0 ? min(x.len + per, cap) : 0));
  int step = 6;
  while (most >> step >= 128) ++step;
  const auto more = [&](int i) {  // the lane's row tiles that see more than i << step keys
    const int64_t keys = static_cast<int64_t>(i) << step;
    const int64_t rest = keys - prefix;
    const int seen = static_cast<int>(
        min(max(grows ? rest * p.group >> 7 : (rest < 0 ? 0 : int64_t{n_rt}), int64_t{0}),
            static_cast<int64_t>(n_rt)));
    return i < 0 ? n_rt : keys >= cap ? 0 : n_rt - seen;
  };
  const auto all = [&](int n) {
    return __builtin_amdgcn_readlane(wave_scan32(n), 63) * p.num_kv_heads;
  };
  int lo = -1, hi = (most >> step) + 1;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (all(more(mid)) > at) lo = mid;
    else hi = mid;
  }
  const int above = more(hi), here = more(lo) - above;
  const int32_t nth = at - all(above);
  const int incl = wave_scan32(here) * p.num_kv_heads;
  const int j = __builtin_amdgcn_readfirstlane(
      min(static_cast<int>(__popcll(__ballot(incl <= nth))), 63));
  const int in = nth - (j > 0 ? __builtin_amdgcn_readlane(incl, j - 1) : 0);
  P16Group gr;
  gr.r = __builtin_amdgcn_readfirstlane(min(j, p.num_reqs - 1));
  gr.req = p16_request_of<kP16WideRows>(p, gr.r, __builtin_amdgcn_readlane(c.of.q0, j),
                                        __builtin_amdgcn_readlane(c.of.q1, j),
                                        __builtin_amdgcn_readlane(c.of.len, j));
  gr.group = gr.kt = gr.number = 0;
  const int before = __builtin_amdgcn_readlane(above, j);
  const int k = static_cast<int>(static_cast<uint32_t>(in) / static_cast<uint32_t>(p.num_kv_heads));
  u.head = __builtin_amdgcn_readfirstlane(in - k * p.num_kv_heads);
  u.rt = __builtin_amdgcn_readfirstlane(max(gr.req.n_rt - 1 - before - k, 0));
  return gr;
}

template <int D, bool kF16>
__global__ __launch_bounds__(64 * kP16Waves, WideOf<D>::kPerSimd) void f8_wide(
    const F8Params p) {
  using W = WideOf<D>;
  constexpr int kBM = kP16WideRows, kKT = kP16WideKeys;
  constexpr float kSlack = 8.0f, kBias = 16.0f;
  __shared__ __attribute__((aligned(16))) char lds[4 * W::kBuf];  // K, K, V, V
  __shared__ F8Window s_window[kP16Waves];
  __shared__ int32_t s_nan[2][kP16Waves];
  __shared__ float s_scale[2][kP16Waves];
  __shared__ uint16_t s_bad[W::kO][64 * kP16Waves];  // columns that a row's NaN is in

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r32 = lane & 31, h = lane >> 5;
  P16Cursor cur;
  const int64_t tiles = p16_begin<kBM>(p, cur, lane);
  const int takers = p16_takers(p, tiles);
  // Where groups are cut, the work-groups of an XCD (every eighth) take neighbouring
  // shares, so that the row tiles of one KV head read its keys from one L2; those without
  // a share are last, in each XCD alike.
  const bool cuts = p.notes >= 0;
  int wg = blockIdx.x;
  if (cuts && (p.num_wg & 7) == 0) {
    const int per = (takers + 7) >> 3, xcd = wg & 7, nth = wg >> 3;
    wg = nth < per ? xcd * per + nth : wg;
  }
  if (wg == 0) p16_note_groups<kBM, D>(p, cur, lane);
  if (wg >= takers) {
    if (threadIdx.x == 0) p16_note_none<D>(p, wg);
    return;
  }
  int64_t at = p16_share(tiles, wg, takers);
  const int64_t end = p16_share(tiles, wg + 1, takers);
  bool noted = false;

  while (at < end) {
    P16Unit u;
    P16Group gr;
    if (cuts || p.num_reqs > 64 || p.key_tile_log2 < W::kSort) {
      gr = p16_locate<kBM>(p, cur, at, lane);
      u = p16_unit(gr.req, gr.group);
      if (!cuts) {  // a request's last row tiles first, in turn the KV heads of each
        const uint32_t heads = static_cast<uint32_t>(p.num_kv_heads);
        u.rt = static_cast<int32_t>(static_cast<uint32_t>(gr.group) / heads);
        u.head = gr.group - u.rt * static_cast<int32_t>(heads);
        u.rt = gr.req.n_rt - 1 - u.rt;
      }
    } else {
      gr = f8_longest(p, cur, static_cast<int32_t>(at), lane, u);
    }
    const int take = static_cast<int>(min(static_cast<int64_t>(gr.req.n_kt - gr.kt), end - at));
    const bool whole = take == gr.req.n_kt;
    const int slot = 2 * wg + (gr.kt == 0 ? 1 : 0);
    const int rows = min(kBM, gr.req.rows - u.rt * kBM);
    const int row = 32 * wave + r32;
    const bool live = row < rows;
    int64_t token, head;
    p16_row<kBM>(p, gr.req.q0, u, min(row, rows - 1), token, head);

    // The lane's row sees the keys before row_hi, of them its window. The piece's 64-key tiles
    // [t0, t1) from base on, of those that the unit sees any key of; those of them in
    // [full0, full1) are seen whole by all rows of the unit, those outside of
    // [w0, w1) by none of the wave's, and those in [wf0, wf1) whole by all of these.
    const int len = gr.req.len, base = gr.req.base;
    const bool idle = 32 * wave >= rows;  // a wave without rows only loads
    int row_hi = len;
    int t0 = 0, t1, full0, full1, w0, w1, wf0, wf1;
    {
      const int n = p.qsl == nullptr
                        ? 1
                        : static_cast<int>(p.g_div.div(static_cast<uint32_t>(gr.req.rows)));
      const auto hi_of = [&](int t) { return p.causal ? max(len - (n - 1 - t), 0) : len; };
      const auto lo_of = [&](int hi) { return p.window > 0 ? max(hi - p.window, 0) : 0; };
      const auto token_of = [&](int r) {
        return static_cast<int>(p.g_div.div(
            static_cast<uint32_t>(u.rt * kBM + min(r, rows - 1))));
      };
      row_hi = hi_of(static_cast<int>(token) - gr.req.q0);
      // First tile of the keys from `key` on, and one past the last of those before.
      const auto down = [&](int key) { return key > base ? (key - base) >> 6 : 0; };
      const auto up = [&](int key) { return key > base ? (key - base + kKT - 1) >> 6 : 0; };
      const auto uniform = [](int x) { return __builtin_amdgcn_readfirstlane(x); };
      const int u_first = hi_of(token_of(0)), u_last = hi_of(token_of(kBM - 1));
      const int w_first = hi_of(token_of(32 * wave)), w_last = hi_of(token_of(32 * wave + 31));
      const int log = p.key_tile_log2 - 6;
      // A piece is tiles of those that the unit sees; whole ones are one "tile".
      const int first = down(lo_of(u_first)), last = up(u_last);
      t0 = uniform(first + (whole ? 0 : gr.kt << log));
      t1 = uniform(whole ? last : min(first + ((gr.kt + take) << log), last));
      full0 = uniform(up(lo_of(u_last)));
      full1 = uniform(down(u_first));
      w0 = uniform(idle ? INT32_MAX : down(lo_of(w_first)));
      w1 = uniform(up(w_last));
      wf0 = uniform(up(lo_of(w_last)));
      wf1 = uniform(down(w_first));
    }

    const auto row_lo_of = [&] { return p.window > 0 ? max(row_hi - p.window, 0) : 0; };

    float m = kNegInf, l = 0.0f;
    bool bad = false;
    f32x16 o[W::kO];
#pragma unroll
    for (int j = 0; j < W::kO; ++j)
#pragma unroll
      for (int i = 0; i < 16; ++i) o[j][i] = 0.0f;

    const int32_t* table = p.block_table + static_cast<int64_t>(gr.r) * p.bt_stride;
    // Entry i of the wave's window: the block of 16 keys that it brings of tile
    // window + i.
    int window = t0;
    const auto refill = [&](int t) {
      window = t;
      const F8Block b = f8_block(p, table, u.head, f8_tile_block(base, t + lane, wave, len));
      s_window[wave].address[lane] =
          (u32x4){static_cast<uint32_t>(b.k), static_cast<uint32_t>(b.k >> 32),
                  static_cast<uint32_t>(b.v), static_cast<uint32_t>(b.v >> 32)};
      s_window[wave].e[lane] = b.e;
    };
    // Lane: 16 codes from column 16 c on of row r and of every kStep-th after it.
    constexpr int kStep = 64 / W::kCodes;
    const int r0 = lane / W::kCodes, c0 = lane % W::kCodes;
    typedef u32x4 __attribute__((address_space(1))) GlobalPiece;
    u32x4 kc[W::kLoads], vc[W::kLoads];
    uint32_t ke = 0, ve = 0;
    u32x4 found = {0u, 0u, 0u, 0u};
    uint32_t found_e = 0;
    const auto find = [&](int t) {
      found = s_window[wave].address[t - window];
      found_e = s_window[wave].e[t - window];
    };
    const auto load = [&](int t) {
      const int at_lane = t - window;
      const u32x4 address = W::kEarly ? found : s_window[wave].address[at_lane];
      const GlobalBytes ks = f8_uniform(address[0], address[1]);
      const GlobalBytes vs = f8_uniform(address[2], address[3]);
      const uint32_t e = __builtin_amdgcn_readfirstlane(W::kEarly ? found_e
                                                                  : s_window[wave].e[at_lane]);
      ke = e & 0xffu;
      ve = e >> 8;
      const uint32_t k_slot = static_cast<uint32_t>(p.k.s_slot);
      const uint32_t v_slot = static_cast<uint32_t>(p.v.s_slot);
      const uint32_t ko = __umul24(r0, k_slot) + 16 * c0, vo = __umul24(r0, v_slot) + 16 * c0;
#pragma unroll
      for (int i = 0; i < W::kLoads; ++i) {
        kc[i] = *reinterpret_cast<const GlobalPiece*>(
            ks + static_cast<int64_t>(i * kStep) * k_slot + ko);
        vc[i] = *reinterpret_cast<const GlobalPiece*>(
            vs + static_cast<int64_t>(i * kStep) * v_slot + vo);
      }
    };
    // Part `part` of four of the loaded tile into buffer `buf`. The pieces' places
    // differ in bits that an exclusive or or an addition sets.
    const auto store = [&](int buf, int part) {
      char* kd = lds + buf * W::kBuf + 16 * wave * W::kRow;
      char* vd = kd + 2 * W::kBuf;
      const uint32_t ka = r0 * W::kRow + 16 * W::k_piece(r0, 2 * c0);
      const uint32_t va = r0 * W::kRow + 16 * W::v_piece(r0, 2 * c0);
#pragma unroll
      for (int q = 0; q < W::kLoads; ++q) {
        const int at = part * W::kLoads + q, i = (at >> 1) % W::kLoads, e = at & 1;
        if (at < 2 * W::kLoads)
          *reinterpret_cast<u32x4*>(kd + (ka ^ (W::kOddK * e) ^ W::k_row(i)) +
                                    kStep * i * W::kRow) =
              f8_eight<kF16>(kc[i][2 * e], kc[i][2 * e + 1], kF16 ? 1.0f : f8_scale(ke));
        else
          *reinterpret_cast<u32x4*>(vd + (va ^ (W::kOddV * e)) + kStep * i * W::kRow) =
              f8_eight<false>(vc[i][2 * e], vc[i][2 * e + 1], f8_scale(ve));
      }
    };
    // What the others have to know of it: whether there is a NaN in V, where not
    // all rows see all of tile t; the scale of K's block, in fp16.
    const auto tell = [&](int t, int buf) {
      if (__builtin_expect(t < full0 || t >= full1, 0)) {
        bool any = false;
#pragma unroll
        for (int i = 0; i < W::kLoads; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) any |= f8_has_nan(vc[i][e]);
        const bool nan = __ballot(any) != 0;
        if (lane == 0) s_nan[buf][wave] = nan;
      }
      if (kF16 && lane == 0) s_scale[buf][wave] = f8_scale(ke);
    };
    const auto store_all = [&](int t, int buf) {
#pragma unroll
      for (int part = 0; part < 4; ++part) store(buf, part);
      tell(t, buf);
    };

    int buf = 0;
    lds_barrier();  // the last unit's reads of both buffers are done
    if (t0 < t1) {
      refill(t0);
      if constexpr (W::kEarly) find(t0);
      load(t0);
    }
    u32x4 q[W::kQ];
    {
      const char* src = p.q + token * p.s_q_tok + head * p.s_q_head + 16 * h;
#pragma unroll
      for (int j = 0; j < W::kQ; ++j) {
        q[j] = *reinterpret_cast<const u32x4*>(src + 32 * j);
        if (!live) q[j] = (u32x4){0u, 0u, 0u, 0u};
      }
    }
    if (gr.kt == 0 && (!whole || p.notes > 0)) {
      noted |= !whole;
      if (threadIdx.x == 0) p16_note<D>(p, gr, wg, tiles, at, takers, !whole);
    }
    at += take;
    if (t0 < t1) store_all(t0, 0);

    for (int t = t0; t < t1; ++t, buf ^= 1) {
      lds_barrier();  // tile t is in LDS, and nobody reads tile t - 1 any more
      const bool more = t + 1 < t1;
      const int k0 = base + kKT * t;
      const char* kt = lds + buf * W::kBuf;
      const char* vt = kt + 2 * W::kBuf;
      const bool masked = t < full0 || t >= full1;
      if (__builtin_expect(masked && (s_nan[buf][0] | s_nan[buf][1] | s_nan[buf][2] |
                                      s_nan[buf][3]) != 0, 0)) {
        // A NaN in V that not all rows see: the lane's columns of which its row sees
        // one are noted, and the tile is rid of them.
#pragma unroll 1
        for (int j = 0; j < W::kO; ++j) {
          uint32_t bits = 0;
#pragma unroll 1
          for (int k = 0; k < kKT; ++k) {
            const bool sees = k0 + k >= row_lo_of() && k0 + k < row_hi;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const int col = 32 * j + 8 * (i >> 2) + 4 * h + (i & 3);
              const uint16_t w = *reinterpret_cast<const uint16_t*>(
                  vt + k * W::kRow + 16 * W::v_piece(k & 15, col >> 3) + 2 * (col & 7));
              bits |= sees && (w & 0x7fffu) > 0x7f80u ? 1u << i : 0u;
            }
          }
          s_bad[j][threadIdx.x] = static_cast<uint16_t>(bits | (bad ? s_bad[j][threadIdx.x] : 0u));
        }
        bad = true;
        lds_barrier();
        char* vd = lds + (buf + 2) * W::kBuf + 16 * wave * W::kRow;
#pragma unroll
        for (int i = 0; i < W::kRow / 64; ++i) {
          u32x4* x = reinterpret_cast<u32x4*>(vd + 1024 * i + 16 * lane);
          u32x4 y = *x;
#pragma unroll
          for (int e = 0; e < 4; ++e) y[e] = f8_without_nan(y[e]);
          *x = y;
        }
        lds_barrier();
      }
      const bool mine = t >= w0 && t < w1;
      if (__builtin_expect(more && t + 1 - window == 64, 0)) refill(t + 1);
      if (W::kEarly && more) find(t + 1);
      if (more && !mine) {
        load(t + 1);
        store_all(t + 1, buf ^ 1);
      }
      if (mine) {
        // Scores: K operands four products ahead.
        f32x16 s[2];
        u32x4 kf[2][4];
        const auto read_k = [&](int n) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int b = e & 1, j = 2 * n + (e >> 1);
            kf[n & 1][e] = *reinterpret_cast<const u32x4*>(kt + (32 * b + r32) * W::kRow +
                                                           16 * W::k_piece(r32, 2 * j + h));
          }
        };
        read_k(0);
#pragma unroll
        for (int n = 0; n < W::kQ / 2; ++n) {
          if (n + 1 < W::kQ / 2) read_k(n + 1);
          __builtin_amdgcn_sched_barrier(0);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int b = e & 1, j = 2 * n + (e >> 1);
            if (j == 0)
#pragma unroll
              for (int i = 0; i < 16; ++i) s[b][i] = 0.0f;
            s[b] = mfma32<kF16>(kf[n & 1][e], q[j], s[b]);
          }
          __builtin_amdgcn_sched_barrier(0);
        }
        // V operands of 16 keys: rows 16 i + 4 h + 0..3 and 8 further on, columns
        // 32 j + l % 32.
        u32x4 vf[2][W::kO];
        const auto read_v = [&](int i) {
          const int r0 = 4 * h + ((lane & 15) >> 2);
#pragma unroll
          for (int j = 0; j < W::kO; ++j) {
            const int byte = 64 * j + 32 * ((lane >> 4) & 1) + 8 * (lane & 3);
            const char* a =
                vt + (16 * i + r0) * W::kRow + 16 * W::v_piece(r0, byte >> 4) + (byte & 15);
            const u32x2 x = column4(a), y = column4(a + 8 * W::kRow);
            vf[i & 1][j] = (u32x4){x[0], x[1], y[0], y[1]};
          }
        };
        // The next tile is on its way during the softmax and the PV products, in the
        // registers that K's operands had.
        if (more) load(t + 1);
        // The softmax goes before the products of the SIMD's other waves.
        __builtin_amdgcn_s_setprio(2);
        read_v(0);
        if constexpr (kF16) {
#pragma unroll
          for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int i = 0; i < 16; ++i) s[b][i] *= s_scale[buf][2 * b + (i >> 3)];
        }
        if (__builtin_expect(t < wf0 || t >= wf1, 0)) {
          const int row_lo = row_lo_of();
#pragma unroll
          for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const int key = k0 + 32 * b + 8 * (i >> 2) + 4 * h + (i & 3);
              s[b][i] = key >= row_lo && key < row_hi ? s[b][i] : kNegInf;
            }
        }
        float top = fmaxf(s[1][15], s[0][15]);
#pragma unroll
        for (int i = 0; i < 15; ++i) top = max3_raw(top, s[0][i], s[1][i]);
        {
          const SwapPair sw = swap_halves(top);
          top = max_raw(sw.a, sw.b) * p.scale_log2;
        }
        if (__ballot(top > m + kSlack) != 0) {
          const float next = fmaxf(m, top);
          const float ref = next == kNegInf ? 0.0f : next;
          float alpha = __builtin_amdgcn_exp2f(m - ref);
          m = next;
          // In place, as p16_wide.hip: otherwise the branch costs a copy of O in
          // every tile. The first product needs a wait after the exp2; O's own
          // products were issued before the scores'.
          asm volatile("s_nop 3" : "+v"(alpha));
          l *= alpha;
#pragma unroll
          for (int j = 0; j < W::kO; ++j)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              float x = o[j][i];
              asm volatile("v_mul_f32 %0, %0, %1" : "+v"(x) : "v"(alpha));
              o[j][i] = x;
            }
        }
        const float shift = (m == kNegInf ? 0.0f : m) + kBias;
        u32x4 pf[4], pl[kF16 ? 4 : 1];
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
          for (int i = 0; i < 16; i += 2) {
            const float x0 = __builtin_amdgcn_exp2f(s[b][i] * p.scale_log2 - shift);
            const float x1 = __builtin_amdgcn_exp2f(s[b][i + 1] * p.scale_log2 - shift);
            const uint32_t w = pack16<false>(x0, x1);
            pf[2 * b + (i >> 3)][(i & 7) >> 1] = w;
            if constexpr (kF16) {
              l += x0;
              l += x1;
              pl[2 * b + (i >> 3)][(i & 7) >> 1] =
                  pack16<false>(x0 - __builtin_bit_cast(float, w << 16),
                                x1 - __builtin_bit_cast(float, w & 0xffff0000u));
            } else {
              l = add_pair<false>(w, l);
            }
          }
        __builtin_amdgcn_s_setprio(0);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          __builtin_amdgcn_sched_barrier(0);
          // The first operands, read before the softmax, are waited for before the
          // next ones are asked for, and not with them.
          if (i == 0) __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0)
          if (i < 3) read_v(i + 1);
          __builtin_amdgcn_sched_barrier(0);
#pragma unroll
          for (int j = 0; j < W::kO; ++j) {
            o[j] = mfma32<false>(vf[i & 1][j], pf[i], o[j]);
            if constexpr (kF16) o[j] = mfma32<false>(vf[i & 1][j], pl[i], o[j]);
          }
          // Behind the last tile, the registers' old codes, which nobody reads.
          store(buf ^ 1, i);
        }
        if (more) tell(t + 1, buf ^ 1);
        __builtin_amdgcn_s_setprio(1);
      }
    }

    if (bad) {
#pragma unroll
      for (int j = 0; j < W::kO; ++j) {
        const uint32_t bits = s_bad[j][threadIdx.x];
#pragma unroll
        for (int i = 0; i < 16; ++i) o[j][i] = bits >> i & 1u ? __builtin_nanf("") : o[j][i];
      }
    }
    {
      // The row's place again, rather than in registers through the loop.
      int again = min(row, rows - 1);
      asm volatile("" : "+v"(again));
      p16_row<kBM>(p, gr.req.q0, u, again, token, head);
    }
    const SwapPair ls = swap_halves(l);
    const float sum = ls.a + ls.b;
    if (live && !whole) {
      float* dst = p16_slot_o<D>(p, slot, 0, row) + 4 * h;
#pragma unroll
      for (int j = 0; j < W::kO; ++j)
#pragma unroll
        for (int b = 0; b < 4; ++b)
          *reinterpret_cast<f32x4*>(dst + 32 * j + 8 * b) =
              (f32x4){o[j][4 * b], o[j][4 * b + 1], o[j][4 * b + 2], o[j][4 * b + 3]};
      if (h == 0) *reinterpret_cast<f32x2*>(p16_slot_ml<D>(p, slot, 0, row)) = (f32x2){m, sum};
    } else if (live) {
      const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
      char* dst = p.out + token * p.s_out_tok + head * p.s_out_head + 8 * h;
#pragma unroll
      for (int j = 0; j < W::kO; ++j)
#pragma unroll
        for (int b = 0; b < 4; ++b)
          *reinterpret_cast<u32x2*>(dst + 64 * j + 16 * b) =
              (u32x2){pack16<kF16>(o[j][4 * b] * inv, o[j][4 * b + 1] * inv),
                      pack16<kF16>(o[j][4 * b + 2] * inv, o[j][4 * b + 3] * inv)};
    }
  }
  if (!noted && threadIdx.x == 0) p16_note_none<D>(p, wg);
}

}  // namespace

hipError_t launch_f8_wide_kernel(const F8Params& p, bool f16, int head_size, hipStream_t stream) {
  note_kernel("f8_wide");
  const dim3 grid(static_cast<unsigned>(p.num_wg)), block(64 * kP16Waves);
  switch (head_size) {
    case 64:
      if (f16) f8_wide<64, true><<<grid, block, 0, stream>>>(p);
      else f8_wide<64, false><<<grid, block, 0, stream>>>(p);
      break;
    case 256:
      if (f16) f8_wide<256, true><<<grid, block, 0, stream>>>(p);
      else f8_wide<256, false><<<grid, block, 0, stream>>>(p);
      break;
    default:
      if (f16) f8_wide<128, true><<<grid, block, 0, stream>>>(p);
      else f8_wide<128, false><<<grid, block, 0, stream>>>(p);
  }
  return hipGetLastError();
}

}  // namespace pa
