// p16_rows.hip -- attention of few query rows over a paged 16-bit cache: one
// new token per request, or the few decoder tokens that attend to an
// encoder's states. A unit is 16 rows of one KV head (p16.h); its keys go
// through the four waves of a work-group in turn, 32 at a time, each wave with
// its own running maximum m and sum l of the online softmax
//   m' = max(m, s), l' = l 2^(m - m') + sum 2^(s - m'), o' = o 2^(m - m') + 2^(s - m') v
// (s in units of log2), which the work-group joins at the end of the unit.
//
// Layout. Nothing goes through LDS before that end. v_mfma_f32_16x16x32 with
// the keys on M and the query rows on N: K's operand is 16 bytes of a key row
// per lane as the cache holds it (lane l: key l % 16, values 8 (l / 16) + 32 j),
// and lane l gets the scores of query row l % 16 for the keys
// 16 b + 4 (l / 16) + i of the 32. Those are the B operand of the PV product as
// they are, if V takes the same keys in the same order: lane l loads 16 bytes
// (the 8 columns from 8 (l % 16) on; 4 at D = 64) of each of those eight key
// rows, whole rows per load, and an 8 x 8 transposition in registers (one
// v_perm_b32 per two values) makes the operand of each of the 8 columns.
//
// Pipeline. The next chunk's K is loaded when its registers are free, after
// the QK products, its V after the PV products; its page numbers, read on the
// scalar unit, a chunk before. So a wave always has 4 to 16 KB in flight.
//
// Numerics. Scores, m, l and o are 32 bits. P is a 16-bit pair hi + lo (16 to
// 22 significant bits, in fp16 scaled by 2^14 for its short range): the second
// product costs matrix time that this kernel has to spare, being bound by the
// cache's bytes. A masked key takes the
// address of a visible one and the weight 0, so nothing behind a request's
// last key, or in another's page, can reach a sum, whatever it holds.
//
// Bound: the cache's bytes, each read once, by one work-group. 64 requests of
// 1,024 to 32,768 keys (32q / 8kv of 128, bf16, 4.20 GB): 625 us, 6.7 TB/s, and
// the fabric counters see 4.21 GB. On the way there, same call: plain loads
// 757 us; non-temporal ones 709; the KV heads of NHD pages side by side in a
// work-group, which so reads whole slots, 656; one work-group per compute unit
// instead of two 626. MFMA is busy 7 % of the SIMDs' time, VALU 17 %. At short
// lengths the bound is latency, of four dependent reads (lengths, page number,
// K, the join's): one request to 1,024 keys 6.9 us + 2.5 of join, 16 windows of
// 4,096 keys at D = 256 29.2 us (4.6 TB/s).

#include <type_traits>

#include "p16_device.h"

namespace pa {
namespace {

template <int D>
struct RowsDim {
  static constexpr int kQ = D / 32;                  // QK products per 16 keys
  static constexpr int kCols = D < 128 ? D / 16 : 8; // columns per V load
  static constexpr int kPieces = D / (16 * kCols);   // V loads per key row
  static constexpr int kO = D / 16;                  // PV products per chunk
  static constexpr int kPerSimd = p16_resident(D);   // a work-group has a wave on each SIMD
  // At D = 256 the registers do not hold Q beside K, V and O.
  static constexpr bool kQInLds = D == 256;
};

template <int kCols>
struct VRun;
template <>
struct VRun<4> { typedef u32x2 type; };
template <>
struct VRun<8> { typedef u32x4 type; };

template <bool kF16>
__device__ __forceinline__ float low16(uint32_t w) {
  if constexpr (kF16) return static_cast<float>(__builtin_bit_cast(f16x2, w)[0]);
  else return __builtin_bit_cast(float, w << 16);
}
template <bool kF16>
__device__ __forceinline__ float high16(uint32_t w) {
  if constexpr (kF16) {
    const uint32_t h = w >> 16;
    return static_cast<float>(__builtin_bit_cast(f16x2, h)[0]);
  } else {
    return __builtin_bit_cast(float, w & 0xffff0000u);
  }
}

// The keys of a unit in 16-key blocks as a lane addresses them: with pages of
// a multiple of 16 slots (kPage16), one page per block, its number read on the
// scalar unit, and offsets within the block that a wave keeps; otherwise one
// page per key.
template <bool kPage16>
struct Walker {
  const P16Params& p;
  const int32_t* table;  // the request's row of the block table
  int32_t lo, len;       // visible keys
  int64_t head;

  // A block whose rows are all in the cache's pages.
  struct Block {
    int32_t kb;
    const char *k, *v;  // its first rows (kPage16)
  };
  __device__ __forceinline__ int32_t valid(int32_t id) const {
    return static_cast<uint32_t>(id) < static_cast<uint32_t>(p.num_blocks) ? id : 0;
  }
  // The block that stands for the 16 keys from k0 on: itself, or the last one.
  __device__ __forceinline__ int32_t start(int32_t k0) const { return min(k0, (len - 1) & ~15); }
  // Its entry of the block table, and the block itself.
  __device__ __forceinline__ uint32_t page_of(int32_t kb) const {
    return mulhi32(static_cast<uint32_t>(kb), p.bs_div.mul) >> p.bs_div.shift;  // block size > 1
  }
  __device__ __forceinline__ int32_t entry(int32_t k0) const {
    return kPage16 ? ld_ro(table, page_of(start(k0))) : 0;
  }
  __device__ __forceinline__ Block block(int32_t k0, int32_t entry) const {
    Block b;
    b.kb = start(k0);
    if constexpr (kPage16) {
      const int64_t id = valid(entry);
      const int64_t first = b.kb - static_cast<int32_t>(page_of(b.kb) * p.bs_div.d);
      b.k = p.k.base + id * p.k.s_block + first * p.k.s_slot + head * p.k.s_head;
      b.v = p.v.base + id * p.v.s_block + first * p.v.s_slot + head * p.v.s_head;
    }
    return b;
  }
  // Byte `col` of row i of the block in stream s, brought into the visible keys.
  __device__ __forceinline__ const char* row(const CacheStream& s, const char* first, int32_t kb,
                                             int32_t i, int32_t col) const {
    const int32_t at = min(max(i, lo - kb), len - 1 - kb);
    if constexpr (kPage16) {
      return first + (__umul24(static_cast<uint32_t>(at), static_cast<uint32_t>(s.s_slot)) + col);
    } else {
      const uint32_t key = static_cast<uint32_t>(kb + at);
      const uint32_t pg = p.bs_div.div(key);
      return s.base + static_cast<int64_t>(valid(table[pg])) * s.s_block +
             static_cast<int64_t>(key - pg * p.bs_div.d) * s.s_slot + head * s.s_head + col;
    }
  }
};

template <int D, bool kF16, bool kPage16>
__global__ __launch_bounds__(64 * kP16Waves, RowsDim<D>::kPerSimd) void p16_rows(
    const P16Params p) {
  using R = RowsDim<D>;
  using V = typename VRun<R::kCols>::type;
  constexpr int kBM = kP16RowsRows;
  constexpr float kBias = kF16 ? 14.0f : 0.0f;  // P is scaled by 2^kBias
  // The sums of the waves that are not their unit's first, at the end; Q
  // before it, if it lives here.
  __shared__ f32x4 s_x[kP16Waves][R::kO][64];
  __shared__ float s_m[kP16Waves][kBM], s_l[kP16Waves][kBM];

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

    float m = kNegInf, l = 0.0f;
    f32x4 o[R::kO];
#pragma unroll
    for (int j = 0; j < R::kO; ++j) o[j] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};

    Walker<kPage16> w{p, p.block_table + static_cast<int64_t>(gr.r) * p.bt_stride, gr.req.lo,
                      gr.req.len, u.head};
    const int step = 32 * parts;
    const int k_end = min(gr.req.base + ((gr.kt + take) << p.key_tile_log2), gr.req.len);
    int k0 = gr.req.base + (gr.kt << p.key_tile_log2) + 32 * part;

    // The page numbers are on their way while Q is read.
    int32_t first_entry[2] = {0, 0};
    if (k0 < k_end) {
      first_entry[0] = w.entry(k0);
      first_entry[1] = w.entry(k0 + 16);
    }
    // Q: 16 bytes per product, zeros in rows that the unit lacks.
    if (!first && parts > 1) __syncthreads();  // the last group's sums have been read
    first = false;
    u32x4 q[R::kQ];
    {
      const char* src = p.q + token * p.s_q_tok + head * p.s_q_head + 16 * g;
#pragma unroll
      for (int j = 0; j < R::kQ; ++j) {
        q[j] = *reinterpret_cast<const u32x4*>(src + 64 * j);
        if (r16 >= rows) q[j] = (u32x4){0u, 0u, 0u, 0u};
        if constexpr (R::kQInLds) s_x[wave][j][lane] = __builtin_bit_cast(f32x4, q[j]);
      }
    }

    u32x4 kf[2][R::kQ];
    V vf[8][R::kPieces];
    auto load_k = [&](const typename Walker<kPage16>::Block& x, int b) {
      const char* src = w.row(p.k, x.k, x.kb, r16, 16 * g);
#pragma unroll
      for (int j = 0; j < R::kQ; ++j) kf[b][j] = ld_nt<u32x4>(src + 64 * j);
    };
    auto load_v = [&](const typename Walker<kPage16>::Block& x, int b) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const char* src = w.row(p.v, x.v, x.kb, 4 * g + e, 2 * R::kCols * r16);
#pragma unroll
        for (int c = 0; c < R::kPieces; ++c) vf[4 * b + e][c] = ld_nt<V>(src + 256 * c);
      }
    };
    if (k0 < k_end) {
      typename Walker<kPage16>::Block blk[2];
#pragma unroll
      for (int b = 0; b < 2; ++b) blk[b] = w.block(k0 + 16 * b, first_entry[b]);
#pragma unroll
      for (int b = 0; b < 2; ++b) load_k(blk[b], b);
#pragma unroll
      for (int b = 0; b < 2; ++b) load_v(blk[b], b);
      int32_t entry[2] = {w.entry(k0 + step), w.entry(k0 + step + 16)};
      // One chunk. kMore: the next one's loads are issued on the way; a branch
      // around them instead would make every wait below as strict as the
      // branch that issues none, and so wait for them.
      auto chunk = [&](auto more) {
        constexpr bool kMore = decltype(more)::value;
        const int next = k0 + step;
        f32x4 s[2];
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          s[b] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
          for (int j = 0; j < R::kQ; ++j) {
            u32x4 qj = q[j];
            if constexpr (R::kQInLds) qj = __builtin_bit_cast(u32x4, s_x[wave][j][lane]);
            s[b] = mfma16<kF16>(kf[b][j], qj, s[b]);
          }
        }
        if constexpr (kMore) {
#pragma unroll
          for (int b = 0; b < 2; ++b) blk[b] = w.block(next + 16 * b, entry[b]);
#pragma unroll
          for (int b = 0; b < 2; ++b) load_k(blk[b], b);
#pragma unroll
          for (int b = 0; b < 2; ++b) entry[b] = w.entry(next + step + 16 * b);
        }
        float t[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) t[e] = s[e >> 2][e & 3] * p.scale_log2;
        if (k0 < gr.req.lo || k0 + 32 > gr.req.len) {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const int key = k0 + 16 * (e >> 2) + 4 * g + (e & 3);
            t[e] = key >= gr.req.lo && key < gr.req.len ? t[e] : kNegInf;
          }
        }
        float top = fmaxf(fmaxf(fmaxf(t[0], t[1]), fmaxf(t[2], t[3])),
                          fmaxf(fmaxf(t[4], t[5]), fmaxf(t[6], t[7])));
        top = fmaxf(m, xor_max(top));
        const float ref = top == kNegInf ? 0.0f : top;
        const float alpha = __builtin_amdgcn_exp2f(m - ref);
        m = top;
        float x[8];
        l *= alpha;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          x[e] = __builtin_amdgcn_exp2f(t[e] - (ref - kBias));
          l += x[e];
        }
        u32x4 hi, lo;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          hi[e] = pack16<kF16>(x[2 * e], x[2 * e + 1]);
          const uint32_t h = hi[e];
          lo[e] = pack16<kF16>(x[2 * e] - low16<kF16>(h), x[2 * e + 1] - high16<kF16>(h));
        }
#pragma unroll
        for (int j = 0; j < R::kO; ++j) o[j] *= alpha;
#pragma unroll
        for (int c = 0; c < R::kPieces; ++c)
#pragma unroll
          for (int j = 0; j < R::kCols; ++j) {
            u32x4 a;
#pragma unroll
            for (int e = 0; e < 4; ++e)
              a[e] = __builtin_amdgcn_perm(vf[2 * e + 1][c][j >> 1], vf[2 * e][c][j >> 1],
                                           j & 1 ? 0x07060302u : 0x05040100u);
            f32x4& acc = o[c * R::kCols + j];
            acc = mfma16<kF16>(a, hi, acc);
            acc = mfma16<kF16>(a, lo, acc);
          }
        if constexpr (kMore) {
#pragma unroll
          for (int b = 0; b < 2; ++b) load_v(blk[b], b);
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
      // Column of product (c, j), register i: 16 kCols c + kCols (4 g + i) + j.
      if (!whole) {
        float* dst = p16_slot_o<D>(p, slot, sub, r16);
#pragma unroll
        for (int c = 0; c < R::kPieces; ++c)
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < R::kCols; j += 4) {
              const f32x4* x = &o[c * R::kCols + j];
              *reinterpret_cast<f32x4*>(dst + 16 * R::kCols * c + R::kCols * (4 * g + i) + j) =
                  (f32x4){x[0][i], x[1][i], x[2][i], x[3][i]};
            }
        if (g == 0)
          *reinterpret_cast<f32x2*>(p16_slot_ml<D>(p, slot, sub, r16)) = (f32x2){m, l};
      } else {
        // A row without keys is 0; one whose scores are all -inf is 0 / 0, NaN.
        const float inv = 1.0f / l;
        const bool none = gr.req.len == 0;
        char* dst = p.out + token * p.s_out_tok + head * p.s_out_head;
#pragma unroll
        for (int c = 0; c < R::kPieces; ++c)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            V y;
#pragma unroll
            for (int j = 0; j < R::kCols; j += 2)
              y[j / 2] = none ? 0u
                              : pack16<kF16>(o[c * R::kCols + j][i] * inv,
                                             o[c * R::kCols + j + 1][i] * inv);
            *reinterpret_cast<V*>(dst + 2 * (16 * R::kCols * c + R::kCols * (4 * g + i))) = y;
          }
      }
    }
  }
  if (!noted && threadIdx.x == 0) p16_note_none<D>(p, wg);
}

template <int D>
hipError_t rows_kernel(const P16Params& p, bool f16, bool page16, hipStream_t stream) {
  const dim3 grid(static_cast<unsigned>(p.num_wg)), block(64 * kP16Waves);
  if (f16 && page16) hipLaunchKernelGGL((p16_rows<D, true, true>), grid, block, 0, stream, p);
  else if (f16) hipLaunchKernelGGL((p16_rows<D, true, false>), grid, block, 0, stream, p);
  else if (page16) hipLaunchKernelGGL((p16_rows<D, false, true>), grid, block, 0, stream, p);
  else hipLaunchKernelGGL((p16_rows<D, false, false>), grid, block, 0, stream, p);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_p16_rows_kernel(const P16Params& p, bool f16, bool page16, int head_size,
                                  hipStream_t stream) {
  note_kernel("p16_rows");
  switch (head_size) {
    case 64: return rows_kernel<64>(p, f16, page16, stream);
    case 256: return rows_kernel<256>(p, f16, page16, stream);
    default: return rows_kernel<128>(p, f16, page16, stream);
  }
}

}  // namespace pa
