// fp8_rows.hip -- attention of few query rows over a paged cache in 8-bit
// floating point (fp8.h): one new token per request, or the few tokens of a
// draft. A unit is 16 rows of one KV head (p16.h has the partition); its keys go
// through the four waves of a work-group in turn, 64 at a time, each wave with
// its own running maximum m and sum l of the online softmax
//   m' = max(m, s), l' = l 2^(m - m') + sum 2^(s - m'), o' = o 2^(m - m') + 2^(s - m') v
// (s in units of log2), which the work-group joins at the end of the unit.
//
// Layout. v_mfma_f32_16x16x32 with the keys on M and the query rows on N, as
// p16_rows.hip has it; a lane's bytes are codes here. Of 16 keys' K, lane l has
// 16 codes of key l % 16 from column 16 (l / 16) of every 64 on, two products'
// operands; of V, one run of D / 16 columns from (D / 16) (l % 16) on, of each
// of the four keys 4 (l / 16) + i whose weights it gets. A byte permutation puts
// two keys' codes of a column side by side (two columns at once), and the
// conversion, one instruction for two values, makes the operand's word, times
// the block's scale: three instructions for four values. A block of 16 keys has
// one scale, so that both the scale of K, a factor of the scores, and that of V
// are the same for a wave.
//
// Numerics. Scores, m, l and o are 32 bits. K's codes are exact in the queries'
// type and V's scaled values in bf16, whose range they need; P is a bf16 pair
// hi + lo (16 significant bits). A key that a row does not see (behind its own,
// behind the request's last one in its block, before the window) has the weight 0
// there, and where its V is NaN that is taken out of the products and put back into
// the rows that see it.
//
// Bound: the cache's bytes, each read once, by one work-group. 64 requests of 1,024 to
// 32,768 keys, 8 heads of 128: 2.1 GB, 340 us, 6.2 TB/s; one request to 131,072 keys 50
// us, 5.3 TB/s; 48 of 4,096, 8 heads of 64, 52 us, 4.4 TB/s; 16 behind windows of 4,096, 4
// heads of 256, 25 us. Short ones: latency, 6 us for 64 keys and 0.9 for each 64 more of
// a wave, 3 for the join where keys are cut.

#include <type_traits>

#include "fp8_device.h"

namespace pa {
namespace {

template <int D>
struct RowsDim {
  static constexpr int kK = D / 64;        // 16-code loads of a key row
  static constexpr int kQ = D / 32;        // QK products per 16 keys
  static constexpr int kRun = D / 16;      // V columns of a lane
  static constexpr int kWords = kRun / 4;  // their words
  static constexpr int kO = D / 16;        // PV products per 32 keys
  static constexpr int kPerSimd = p16_resident(D);  // a work-group has a wave on each SIMD
};
// P is scaled by 2^-kBias: sums of 2^16 values near the type's largest stay
// within 32 bits.
constexpr float kBias = 16.0f;
constexpr int kChunk = 64, kBlocks = kChunk / kF8Span;

// A load; kOnce: with the non-temporal hint, of cache lines that no other wave reads.
template <class T, bool kOnce>
__device__ __forceinline__ T load_of(GlobalBytes p) {
  typedef T __attribute__((address_space(1))) Global;
  if constexpr (kOnce) return __builtin_nontemporal_load(reinterpret_cast<const Global*>(p));
  else return *reinterpret_cast<const Global*>(p);
}

template <int D, bool kF16, bool kOnce>
__global__ __launch_bounds__(64 * kP16Waves, RowsDim<D>::kPerSimd) void f8_rows(
    const F8Params p) {
  using R = RowsDim<D>;
  using V = typename Words<R::kWords>::type;
  constexpr int kBM = kP16RowsRows;
  // The sums of the waves that are not their unit's first, at the end.
  __shared__ f32x4 s_x[kP16Waves][R::kO][64];
  __shared__ float s_m[kP16Waves][kBM], s_l[kP16Waves][kBM];
  // Of a NaN in V: its keys in a chunk, by column; the outputs of a lane that meet it.
  __shared__ uint64_t s_nan_keys[kP16Waves][D], s_bad[kP16Waves][64];

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r16 = lane & 15, g = lane >> 4;
  const int wg = blockIdx.x;
  // The wave's unit of a group, its place among the unit's waves and their number.
  const int log_team = p.team >> 1;
  const int sub = wave & (p.team - 1), part = wave >> log_team, parts = kP16Waves >> log_team;
  P16Cursor cur;
  const int64_t tiles = p16_begin<kBM>(p, cur, lane);
  if (wg == 0) p16_note_groups<kBM, D>(p, cur, lane);
  const int takers = p16_takers(p, tiles);
  if (wg >= takers) {
    if (threadIdx.x == 0) p16_note_none<D>(p, wg);
    return;
  }
  int64_t at = p16_share(tiles, wg, takers);
  const int64_t end = p16_share(tiles, wg + 1, takers);
  bool first = true, noted = false;

  while (at < end) {
    const P16Group gr = p16_locate<kBM>(p, cur, at, lane);
    const int take = static_cast<int>(min(static_cast<int64_t>(gr.req.n_kt - gr.kt), end - at));
    const bool whole = take == gr.req.n_kt;
    const int slot = 2 * wg + (gr.kt == 0 ? 1 : 0);
    const int64_t begin = at;
    at += take;
    // A group's last units may be missing: their waves repeat the last one
    // and drop it.
    const int index = gr.group * p.team + sub, units = p.num_kv_heads * gr.req.n_rt;
    const P16Unit u = p16_unit(gr.req, min(index, units - 1));
    const int rows = index < units ? min(kBM, gr.req.rows - u.rt * kBM) : 0;
    int64_t token, head;
    p16_row<kBM>(p, gr.req.q0, u, min(r16, max(rows - 1, 0)), token, head);
    // The keys [row_lo, row_hi) that the lane's row sees, and what all rows do.
    const int len = gr.req.len, lo = gr.req.lo;
    int row_lo = lo, row_hi = len, all_lo = lo, all_hi = len;
    if (p.causal && p.qsl != nullptr) {
      const int n = static_cast<int>(p.g_div.div(static_cast<uint32_t>(gr.req.rows)));
      const auto end_of = [&](int t) { return len - (n - 1 - t); };
      const auto lo_of = [&](int t) { return p.window > 0 ? max(end_of(t) - p.window, 0) : 0; };
      const int t = static_cast<int>(token) - gr.req.q0;
      row_hi = max(end_of(t), 0);
      row_lo = lo_of(t);
      const int ta = static_cast<int>(p.g_div.div(static_cast<uint32_t>(u.rt * kBM)));
      const int tb = static_cast<int>(
          p.g_div.div(static_cast<uint32_t>(min(u.rt * kBM + kBM, gr.req.rows) - 1)));
      all_hi = end_of(ta);
      all_lo = lo_of(tb);
    }

    float m = kNegInf, l = 0.0f;
    bool bad = false;
    f32x4 o[R::kO];
#pragma unroll
    for (int j = 0; j < R::kO; ++j) o[j] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};

    const uint64_t k_base = reinterpret_cast<uint64_t>(p.k.base + u.head * p.k.s_head);
    const uint64_t v_base = reinterpret_cast<uint64_t>(p.v.base + u.head * p.v.s_head);
    const int32_t* table = p.block_table + static_cast<int64_t>(gr.r) * p.bt_stride;
    const int step = kChunk * parts;
    const int k_end = min(gr.req.base + ((gr.kt + take) << p.key_tile_log2), len);
    int k0 = gr.req.base + (gr.kt << p.key_tile_log2) + kChunk * part;

    // The chunk's blocks of 16 keys: block b is the one of the keys from k + 16 b on,
    // or the last one, and lane l knows block l % 4. Its entry of the block table is
    // read a chunk before its address is made and its exponents are asked for.
    const auto start = [&](int k) { return min(k + kF8Span * (lane & 3), (len - 1) & ~15); };
    const auto entry_of = [&](int k) {
      return table[mulhi32(static_cast<uint32_t>(start(k)), p.bs_div.mul) >> p.bs_div.shift];
    };
    uint64_t k_at = 0, v_at = 0;
    uint32_t ke = 0, ve = 0;
    const auto place = [&](int k, int32_t entry) {
      const int kb = start(k);
      const uint32_t page = mulhi32(static_cast<uint32_t>(kb), p.bs_div.mul) >> p.bs_div.shift;
      const uint32_t id = static_cast<uint32_t>(entry) < static_cast<uint32_t>(p.num_blocks)
                              ? static_cast<uint32_t>(entry)
                              : 0u;
      const uint32_t in = static_cast<uint32_t>(kb) - page * p.bs_div.d;
      k_at = k_base + id * p.k.s_block + in * static_cast<uint64_t>(p.k.s_slot);
      v_at = v_base + id * p.v.s_block + in * static_cast<uint64_t>(p.v.s_slot);
      const uint32_t e = (id * static_cast<uint32_t>(p.n_sub) + in / kF8Span) *
                             static_cast<uint32_t>(p.num_kv_heads) +
                         static_cast<uint32_t>(u.head);
      ke = p.k_exp[e];
      ve = p.v_exp[e];
    };
    const auto block_at = [](uint64_t at_lane, int b) {
      return reinterpret_cast<GlobalBytes>(
          static_cast<uint64_t>(static_cast<uint32_t>(
              __builtin_amdgcn_readlane(static_cast<uint32_t>(at_lane), b))) |
          static_cast<uint64_t>(static_cast<uint32_t>(
              __builtin_amdgcn_readlane(static_cast<uint32_t>(at_lane >> 32), b)))
              << 32);
    };
    int32_t entry = 0;
    if (k0 < k_end) entry = entry_of(k0);
    // Q: 16 bytes per product, zeros in rows that the unit lacks.
    if (!first && parts > 1) __syncthreads();  // the last group's sums have been read
    first = false;
    u32x4 q[R::kQ];
    {
      const char* src = p.q + token * p.s_q_tok + head * p.s_q_head;
#pragma unroll
      for (int j = 0; j < R::kQ; ++j) {
        // Product 2 i + h has columns 64 i + 16 g + 8 h and seven more.
        q[j] = *reinterpret_cast<const u32x4*>(src + 128 * (j >> 1) + 32 * g + 16 * (j & 1));
        if (r16 >= rows) q[j] = (u32x4){0u, 0u, 0u, 0u};
      }
    }

    u32x4 kf[kBlocks][R::kK];
    V vf[kBlocks][4];
    // The lane's places in a block: of K's row, of V's first one.
    const uint32_t k_off = __umul24(r16, static_cast<uint32_t>(p.k.s_slot)) + 16 * g;
    const uint32_t v_off = __umul24(4 * g, static_cast<uint32_t>(p.v.s_slot)) + R::kRun * r16;
    const auto load_k = [&] {
      uint32_t k_here = k_off;  // here, so that it is added by the load itself
      asm volatile("" : "+v"(k_here));
#pragma unroll
      for (int b = 0; b < kBlocks; ++b) {
        const GlobalBytes src = block_at(k_at, b);
#pragma unroll
        for (int j = 0; j < R::kK; ++j) kf[b][j] = load_of<u32x4, kOnce>(src + k_here + 64 * j);
      }
    };
    const auto load_v = [&] {
      uint32_t v_here = v_off;
      asm volatile("" : "+v"(v_here));
#pragma unroll
      for (int b = 0; b < kBlocks; ++b) {
        const GlobalBytes src = block_at(v_at, b);
#pragma unroll
        for (int e = 0; e < 4; ++e)
          vf[b][e] = load_of<V, kOnce>(src + e * static_cast<uint32_t>(p.v.s_slot) + v_here);
      }
    };
    if (k0 < k_end) {
      place(k0, entry);
      load_k();
      entry = entry_of(k0 + step);
      load_v();
      // One chunk. kMore: the next one's loads are issued on the way.
      const auto chunk = [&](auto more) {
        constexpr bool kMore = decltype(more)::value;
        const int next = k0 + step;
        float ks[kBlocks], vs[kBlocks];
#pragma unroll
        for (int b = 0; b < kBlocks; ++b) {
          ks[b] = f8_scale(__builtin_amdgcn_readlane(ke, b)) * p.scale_log2;
          vs[b] = f8_scale(__builtin_amdgcn_readlane(ve, b));
        }
        f32x4 s[kBlocks];
#pragma unroll
        for (int b = 0; b < kBlocks; ++b) {
          s[b] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
          for (int j = 0; j < R::kQ; ++j) {
            const u32x4 w = kf[b][j >> 1];
            const u32x4 a = j & 1 ? f8_eight<kF16>(w[2], w[3], 1.0f) : f8_eight<kF16>(w[0], w[1], 1.0f);
            s[b] = mfma16<kF16>(a, q[j], s[b]);
          }
        }
        if constexpr (kMore) {
          // Not before the last product, in whose registers they arrive.
          __builtin_amdgcn_sched_barrier(0);
          place(next, entry);
          load_k();
          entry = entry_of(next + step);
        }
        float t[4 * kBlocks];
#pragma unroll
        for (int e = 0; e < 4 * kBlocks; ++e) t[e] = s[e >> 2][e & 3] * ks[e >> 2];
        const bool edge = k0 < all_lo || k0 + kChunk > all_hi;
        if (__builtin_expect(edge, 0)) {
#pragma unroll
          for (int e = 0; e < 4 * kBlocks; ++e) {
            const int key = k0 + 16 * (e >> 2) + 4 * g + (e & 3);
            t[e] = key >= row_lo && key < row_hi ? t[e] : kNegInf;
          }
        }
        float top = m;
#pragma unroll
        for (int e = 0; e < 4 * kBlocks; ++e) top = fmaxf(top, t[e]);
        top = xor_max(top);
        const float ref = top == kNegInf ? 0.0f : top;
        const float alpha = __builtin_amdgcn_exp2f(m - ref);
        m = top;
        l *= alpha;
        u32x4 hi[kBlocks / 2], lo_[kBlocks / 2];
#pragma unroll
        for (int e = 0; e < 4 * kBlocks; e += 2) {
          const float x = __builtin_amdgcn_exp2f(t[e] - (ref + kBias));
          const float y = __builtin_amdgcn_exp2f(t[e + 1] - (ref + kBias));
          l += x;
          l += y;
          const uint32_t h = pack16<false>(x, y);
          hi[e >> 3][(e & 7) >> 1] = h;
          lo_[e >> 3][(e & 7) >> 1] = pack16<false>(
              x - __builtin_bit_cast(float, h << 16), y - __builtin_bit_cast(float, h & 0xffff0000u));
        }
#pragma unroll
        for (int j = 0; j < R::kO; ++j) o[j] *= alpha;
        // Whether a row may meet a NaN of a key that it does not see.
        bool nan = false;
        if (__builtin_expect(edge, 0)) {
          // Kept in the branch: V is still on its way, and nothing else asks for it here.
          asm volatile("" ::: "memory");
          bool any = false;
#pragma unroll
          for (int b = 0; b < kBlocks; ++b)
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
              for (int i = 0; i < R::kWords; ++i) any |= f8_has_nan(word(vf[b][e], i));
          nan = __ballot(any) != 0;
        }
        // Products of 32 keys, two columns of a word (its low or its high half) at a
        // time; kClean: without NaNs. (V is not changed: the registers' copies would
        // wait for it before the softmax, in chunks that have none, too.)
        const auto pv = [&](auto clean) {
          constexpr bool kClean = decltype(clean)::value;
          const auto codes = [&](int b, int e, int i) {
            const uint32_t w = word(vf[b][e], i);
            return kClean ? w & ~((f8_nan_bytes(w) >> 7) * 0xffu) : w;
          };
#pragma unroll
          for (int h = 0; h < kBlocks / 2; ++h)
#pragma unroll
            for (int i = 0; i < R::kWords; ++i)
#pragma unroll
              for (int c = 0; c < 2; ++c) {
                u32x4 a[2];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                  const int b = 2 * h + (e >> 1);
                  const uint32_t w =
                      __builtin_amdgcn_perm(codes(b, 2 * (e & 1) + 1, i), codes(b, 2 * (e & 1), i),
                                            c ? 0x07030602u : 0x05010400u);
                  a[0][e] = f8_pair_lo<false>(w, vs[b]);
                  a[1][e] = f8_pair_hi<false>(w, vs[b]);
                }
#pragma unroll
                for (int d = 0; d < 2; ++d) {
                  f32x4& acc = o[4 * i + 2 * c + d];
                  acc = mfma16<false>(a[d], hi[h], acc);
                  acc = mfma16<false>(a[d], lo_[h], acc);
                }
              }
        };
        if (__builtin_expect(nan, 0)) {
          // The keys of which a column holds a NaN, as bits; then the columns of the
          // lane's row that see one of them, for the unit's end.
          uint64_t* keys = s_nan_keys[wave];
#pragma unroll
          for (int i = 0; i < D / 64; ++i) keys[64 * i + lane] = 0;
#pragma unroll
          for (int b = 0; b < kBlocks; ++b)
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
              for (int i = 0; i < R::kWords; ++i) {
                const uint32_t w = word(vf[b][e], i), n = f8_nan_bytes(w);
#pragma unroll
                for (int c = 0; c < 4; ++c)
                  atomicOr(reinterpret_cast<unsigned long long*>(&keys[R::kRun * r16 + 4 * i + c]),
                           static_cast<unsigned long long>(n >> (8 * c + 7) & 1u)
                               << (16 * b + 4 * g + e));
              }
          // No branch or loop here differs between lanes. It would change the outer
          // loop's form; and where a loop of a lane's own columns ended, the compiler put
          // the copies that save the walk's registers before the lanes were switched on
          // again (D = 256), so that the next unit was looked up with what lay there.
          const auto before = [](int key) {  // bits of the keys before it
            return key <= 0 ? 0ull : ~0ull >> (64 - min(key, 64));
          };
          const uint64_t sees = before(row_hi - k0) & ~before(row_lo - k0);
          uint64_t hit = bad ? s_bad[wave][lane] : 0;
#pragma unroll 1
          for (int i = 0; i < 4; ++i)
#pragma unroll 1
            for (int j = 0; j < R::kO; ++j)
              hit |= static_cast<uint64_t>((keys[R::kRun * (4 * g + i) + j] & sees) != 0)
                     << (R::kO * i + j);
          s_bad[wave][lane] = hit;
          bad = true;
          pv(std::true_type{});
        } else {
          pv(std::false_type{});
        }
        if constexpr (kMore) {
          __builtin_amdgcn_sched_barrier(0);
          load_v();
          // Unlike the loads before the loop: the compiler would merge both at its
          // head, and copy K and O in every chunk.
          asm volatile("; the next chunk");
          k0 = next;
        }
      };
      while (k0 + step < k_end) chunk(std::true_type{});
      chunk(std::false_type{});
    }

    if (gr.kt == 0 && (!whole || p.notes > 0)) {
      noted |= !whole;
      if (threadIdx.x == 0) p16_note<D>(p, gr, wg, tiles, begin, takers, !whole);
    }
    if (__builtin_expect(bad, 0)) {
      const uint64_t hit = s_bad[wave][lane];
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < R::kO; ++j)
          o[j][i] = hit >> (R::kO * i + j) & 1 ? __builtin_nanf("") : o[j][i];
    }
    // The unit's first wave joins the others' sums to its own.
    l = xor_sum(l);
    if (parts > 1) {
      if (part > 0) {
#pragma unroll
        for (int j = 0; j < R::kO; ++j) s_x[wave][j][lane] = o[j];
        if (g == 0) {
          s_m[wave][r16] = m;
          s_l[wave][r16] = l;
        }
      }
      __syncthreads();
      if (part == 0) {
        for (int v = wave + p.team; v < kP16Waves; v += p.team) {
          const float mv = s_m[v][r16], lv = s_l[v][r16];
          const float top = fmaxf(m, mv);
          const float ref = top == kNegInf ? 0.0f : top;
          const float fa = __builtin_amdgcn_exp2f(m - ref), fb = __builtin_amdgcn_exp2f(mv - ref);
          m = top;
          l = l * fa + lv * fb;
#pragma unroll
          for (int j = 0; j < R::kO; ++j) o[j] = o[j] * fa + s_x[v][j][lane] * fb;
        }
      }
    }
    if (part == 0 && r16 < rows) {
      // The row's place again, rather than in registers through the loop.
      int row = r16;
      asm volatile("" : "+v"(row));
      p16_row<kBM>(p, gr.req.q0, u, row, token, head);
      // Column of product j, register i: kRun (4 g + i) + j.
      if (!whole) {
        float* dst = p16_slot_o<D>(p, slot, sub, r16);
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 0; j < R::kO; j += 4)
            *reinterpret_cast<f32x4*>(dst + R::kRun * (4 * g + i) + j) =
                (f32x4){o[j][i], o[j + 1][i], o[j + 2][i], o[j + 3][i]};
        if (g == 0)
          *reinterpret_cast<f32x2*>(p16_slot_ml<D>(p, slot, sub, r16)) = (f32x2){m, l};
      } else {
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
        char* dst = p.out + token * p.s_out_tok + head * p.s_out_head;
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 0; j < R::kO; j += 4)
            *reinterpret_cast<u32x2*>(dst + 2 * (R::kRun * (4 * g + i) + j)) =
                (u32x2){pack16<kF16>(o[j][i] * inv, o[j + 1][i] * inv),
                        pack16<kF16>(o[j + 2][i] * inv, o[j + 3][i] * inv)};
      }
    }
  }
  if (!noted && threadIdx.x == 0) p16_note_none<D>(p, wg);
}

}  // namespace

hipError_t launch_f8_rows_kernel(const F8Params& p, bool f16, int head_size, hipStream_t stream) {
  note_kernel("f8_rows");
  const dim3 grid(static_cast<unsigned>(p.num_wg)), block(64 * kP16Waves);
  // Two heads of 64 share a cache line where they lie side by side (64 requests of
  // 1,024 to 32,768 keys, 8 heads: NHD pages 246 us with the hint, 210 without; HND
  // pages 180, 198. D = 128 346, 371).
  const auto shared = [&](const CacheStream& s) {
    return p.num_kv_heads > 1 && s.s_head < 128 && s.s_slot > s.s_head;
  };
  const bool once = !(shared(p.k) || shared(p.v));
  switch (head_size) {
    case 64:
      if (f16 && once) f8_rows<64, true, true><<<grid, block, 0, stream>>>(p);
      else if (f16) f8_rows<64, true, false><<<grid, block, 0, stream>>>(p);
      else if (once) f8_rows<64, false, true><<<grid, block, 0, stream>>>(p);
      else f8_rows<64, false, false><<<grid, block, 0, stream>>>(p);
      break;
    case 256:
      if (f16) f8_rows<256, true, true><<<grid, block, 0, stream>>>(p);
      else f8_rows<256, false, true><<<grid, block, 0, stream>>>(p);
      break;
    default:
      if (f16) f8_rows<128, true, true><<<grid, block, 0, stream>>>(p);
      else f8_rows<128, false, true><<<grid, block, 0, stream>>>(p);
  }
  return hipGetLastError();
}

}  // namespace pa
