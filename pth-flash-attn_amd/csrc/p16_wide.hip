// p16_wide.hip -- cross attention of many query rows over a paged 16-bit
// cache: every row of a request sees all of the request's keys. A unit is 128
// rows of one KV head (p16.h), 32 for each of four waves, which share the key
// tiles of 64 in LDS; two work-groups per compute unit (three at D = 64, one at
// D = 256).
//
// Layout. v_mfma_f32_32x32x16 with the keys (or the output columns) on M and
// the wave's query rows on N: lane l holds row l % 32, and of a 32-key score
// tile the keys 8 b + 4 (l / 32) + i (b, i < 4), which are the B operand of the
// PV product as they are if V takes the keys in the same order.
// ds_read_b64_tr_b16 gives a lane one column of four consecutive keys of a
// row-major V, so K and V lie in LDS as in the cache, and come there directly
// (global_load_lds, 16 bytes a lane, a wave 16 keys). A row's 16-byte pieces
// are permuted by the row's number, K's so that 16 consecutive rows' same
// piece, V's so that four consecutive rows' same four pieces lie on different
// banks.
//
// Order of the keys. A group's tiles may be taken in any order, and the
// work-groups of an XCD, which have different row tiles of the same few KV
// heads, take them so that they read the same tile at about the same time:
// after s tiles, a work-group is at tile s modulo the group's number. A whole
// group starts there; of a cut one, the work-group that begins with the rest
// takes the first tiles, and the one that ends with its beginning the last.
//
// Numerics. Scores, m, l and o are 32 bits; the running maximum moves only when
// a score passes it by 2^kSlack, so most tiles rescale nothing. P is rounded
// once to the inputs' type, as the output is: both errors are independent, and
// together sqrt(2) of the output's own; l sums the rounded P, by dot products
// of its pairs. P is scaled by 2^kBias. In bf16 by 2^-kSlack: with the maximum that
// far behind no weight passes 1, so that sums of values near the type's largest
// leave 32 bits no sooner than with the exact maximum. In fp16, whose range is
// short, by 2^12: weights down to 2^-26 of a row's largest keep all 11 bits (2^15
// x 2^16 x 2^31 keys are within 32 bits).
//
// Bound: the matrix cores and the softmax's VALU work, which the SIMD's waves
// run beside each other, at the clock that the power leaves. 4 prompts of 1,500
// to 2,048 rows against 1,601 to 6,404 keys (32q / 8kv of 128, bf16, 6.7e11
// operations), whole call: 652 to 729 us by card, 0.92 to 1.03 PFLOP/s (a library's
// 8192^3 product: 1.2); MFMA is busy 54 % of the time, VALU 46 %, without bank
// conflicts. On the way there: 749 us before the keys' order above (fabric reads
// 3.95 GB, now 0.52), 700 before the waits and priorities below (then 674). 4 x
// 2,048 rows against 4,096 keys (the card of 652): 513 to 519 us, 1.06 PFLOP/s; at
// D = 64 320 to 325 us, 0.85 (the softmax is twice the share); at D = 256, 16q / 8kv,
// 704 to 709 us, 0.78 (one wave per SIMD). No faster, and so not here:
// 256 rows in two halves of four waves that take turns at the matrix cores, a
// tile's PV products between the next one's softmax, a loop of two tiles with
// fixed buffers, staggered starts, and, at D = 64, two tiles on their way instead
// of one (32 rows of 64 requests against 1,500 keys 85.9 -> 91.8 us).

#include "attn_device.h"
#include "p16.h"

namespace pa {
namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef int16_t i16x4 __attribute__((ext_vector_type(4)));

template <int D>
struct WideOf {
  static constexpr int kPerSimd = p16_resident(D);  // a work-group has a wave on each SIMD
  static constexpr int kQ = D / 16;      // QK products per 32 keys
  static constexpr int kO = D / 32;      // output tiles
  static constexpr int kRow = 2 * D;     // bytes of a key row
  static constexpr int kPieces = D / 8;  // 16-byte pieces of a row
  static constexpr int kBuf = kP16WideKeys * kRow;
  static constexpr int kLoads = 16 * kPieces / 64;  // loads of a wave per tile and stream
  // The place of piece c of row t.
  static __device__ __forceinline__ int k_piece(int t, int c) {
    return c ^ (D == 64 ? (t >> 1) & 7 : t & 15);
  }
  static __device__ __forceinline__ int v_piece(int t, int c) {
    return c ^ (D == 64 ? ((t >> 1) & 1) << 2 : (t & 3) << 2);
  }
};

template <bool kF16>
__device__ __forceinline__ f32x16 mfma32(u32x4 a, u32x4 b, f32x16 c) {
  if constexpr (kF16)
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a),
                                                  __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a),
                                                   __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// sum + the two values of a pair.
template <bool kF16>
__device__ __forceinline__ float add_pair(uint32_t w, float sum) {
  if constexpr (kF16)
    return __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2, w),
                                  (f16x2){static_cast<_Float16>(1.0f), static_cast<_Float16>(1.0f)},
                                  sum, false);
  else
    return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, w),
                                           __builtin_bit_cast(bf16x2, 0x3f803f80u), sum, false);
}

// dma16 from a wave's base and 32-bit offsets of its lanes. As a buffer load it
// is not counted with LDS reads, which behind a global one in flight wait for
// all of them at once (D = 256 742 -> 708 us, with column4's restrict).
__device__ __forceinline__ void dma16_from(__amdgpu_buffer_rsrc_t base, uint32_t offset,
                                           char* lds) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(
      base, (void __attribute__((address_space(3)))*)(lds), 16, static_cast<int>(offset), 0, 0, 0);
}
// A buffer of 2 GiB from p on: the callers' offsets are less than 2^29.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer_at(const char* p) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(p), 0, 0x7fffffff, 0x00027000);
}

// A barrier for LDS alone: __syncthreads also waits for stores to memory.
__device__ __forceinline__ void lds_barrier() {
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// Column l % 16 of four rows of a row-major 16-bit matrix in LDS: lane i of
// each 16 gives the address of row i / 4, columns 4 (i % 4). Without restrict
// the compiler has the read wait for every load to LDS in flight, the next
// tile's.
__device__ __forceinline__ u32x2 column4(const char* __restrict__ a) {
  return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                       (i16x4 __attribute__((address_space(3)))*)(
                                           const_cast<char*>(a))));
}

template <int D, bool kF16, bool kPage16>
__global__ __launch_bounds__(64 * kP16Waves, WideOf<D>::kPerSimd) void p16_wide(
    const P16Params p) {
  using W = WideOf<D>;
  constexpr int kBM = kP16WideRows, kKT = kP16WideKeys;
  constexpr float kSlack = kF16 ? 3.0f : 8.0f;
  constexpr float kBias = kF16 ? 12.0f : -kSlack;
  __shared__ __attribute__((aligned(16))) char lds[4 * W::kBuf];  // K, K, V, V

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r32 = lane & 31, h = lane >> 5;
  // The work-groups of an XCD (every eighth) take neighbouring shares, so
  // that the row tiles of one KV head read its keys from one L2.
  const int per = p.num_wg >> 3;
  const int wg = per * 8 == p.num_wg
                     ? static_cast<int>(blockIdx.x & 7) * per + static_cast<int>(blockIdx.x >> 3)
                     : static_cast<int>(blockIdx.x);
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
  bool noted = false;
  uint32_t steps = 0;  // key tiles that this work-group has done

  while (at < end) {
    const P16Group gr = p16_locate<kBM>(p, cur, at, lane);
    const int take = static_cast<int>(min(static_cast<int64_t>(gr.req.n_kt - gr.kt), end - at));
    const bool whole = take == gr.req.n_kt;
    const int slot = 2 * wg + (gr.kt == 0 ? 1 : 0);
    const P16Unit u = p16_unit(gr.req, gr.group);
    const int rows = min(kBM, gr.req.rows - u.rt * kBM);
    const int row = 32 * wave + r32;
    const bool live = row < rows;
    int64_t token, head;
    p16_row<kBM>(p, gr.req.q0, u, min(row, rows - 1), token, head);

    float m = kNegInf, l = 0.0f;
    f32x16 o[W::kO];
#pragma unroll
    for (int j = 0; j < W::kO; ++j)
#pragma unroll
      for (int i = 0; i < 16; ++i) o[j][i] = 0.0f;

    const int32_t* table = p.block_table + static_cast<int64_t>(gr.r) * p.bt_stride;
    const int len = gr.req.len;
    // The lane's bytes within 16 keys, for each load.
    uint32_t k_off[W::kLoads], v_off[W::kLoads];
#pragma unroll
    for (int i = 0; i < W::kLoads; ++i) {
      const int t16 = (64 * i + lane) / W::kPieces, c = (64 * i + lane) % W::kPieces;
      k_off[i] = __umul24(t16, static_cast<uint32_t>(p.k.s_slot)) + 16 * W::k_piece(t16, c);
      v_off[i] = __umul24(t16, static_cast<uint32_t>(p.v.s_slot)) + 16 * W::v_piece(t16, c);
    }
    // The wave's 16 keys of tile t into buffer `buf`; keys past the last
    // one repeat it.
    auto block = [&](int t) { return min(kKT * t + 16 * wave, (len - 1) & ~15); };
    auto page = [&](int t) {  // its entry of the block table
      if constexpr (!kPage16) return 0u;
      return mulhi32(static_cast<uint32_t>(block(t)), p.bs_div.mul) >> p.bs_div.shift;
    };
    auto load = [&](int t, int buf, int32_t entry) {
      const int kb = block(t);
      char* kd = lds + buf * W::kBuf + 16 * wave * W::kRow;
      char* vd = kd + 2 * W::kBuf;
      if constexpr (kPage16) {
        const int64_t id =
            static_cast<uint32_t>(entry) < static_cast<uint32_t>(p.num_blocks) ? entry : 0;
        const int64_t first = kb - static_cast<int32_t>(page(t) * p.bs_div.d);
        const char* ks = p.k.base + id * p.k.s_block + first * p.k.s_slot +
                         static_cast<int64_t>(u.head) * p.k.s_head;
        const char* vs = p.v.base + id * p.v.s_block + first * p.v.s_slot +
                         static_cast<int64_t>(u.head) * p.v.s_head;
        const __amdgpu_buffer_rsrc_t kr = buffer_at(ks), vr = buffer_at(vs);
        if (kb + 16 <= len) {
#pragma unroll
          for (int i = 0; i < W::kLoads; ++i) {
            dma16_from(kr, k_off[i], kd + 1024 * i);
            dma16_from(vr, v_off[i], vd + 1024 * i);
          }
        } else {
#pragma unroll
          for (int i = 0; i < W::kLoads; ++i) {
            const int t16 = (64 * i + lane) / W::kPieces, c = (64 * i + lane) % W::kPieces;
            const uint32_t from = min(t16, len - 1 - kb);
            const uint32_t k_row = __umul24(from, static_cast<uint32_t>(p.k.s_slot));
            const uint32_t v_row = __umul24(from, static_cast<uint32_t>(p.v.s_slot));
            dma16_from(kr, k_row + 16 * W::k_piece(t16, c), kd + 1024 * i);
            dma16_from(vr, v_row + 16 * W::v_piece(t16, c), vd + 1024 * i);
          }
        }
      } else {
#pragma unroll
        for (int i = 0; i < W::kLoads; ++i) {
          const int t16 = (64 * i + lane) / W::kPieces, c = (64 * i + lane) % W::kPieces;
          const uint32_t key = static_cast<uint32_t>(kb + min(t16, len - 1 - kb));
          const uint32_t pg = p.bs_div.div(key);
          int32_t id = table[pg];
          id = static_cast<uint32_t>(id) < static_cast<uint32_t>(p.num_blocks) ? id : 0;
          const int64_t in = static_cast<int64_t>(key - pg * p.bs_div.d);
          const char* ks = p.k.base + static_cast<int64_t>(id) * p.k.s_block + in * p.k.s_slot +
                           static_cast<int64_t>(u.head) * p.k.s_head;
          const char* vs = p.v.base + static_cast<int64_t>(id) * p.v.s_block + in * p.v.s_slot +
                           static_cast<int64_t>(u.head) * p.v.s_head;
          dma16(ks + 16 * W::k_piece(t16, c), kd + 1024 * i);
          dma16(vs + 16 * W::v_piece(t16, c), vd + 1024 * i);
        }
      }
    };

    // The piece's 64-key tiles: `count` of the group's nt from `t_first` on,
    // round its end. Which ones: see the top.
    const int nt = (len + kKT - 1) / kKT;
    const int count = len == 0 ? 0 : gr.req.n_kt == nt ? take : nt;
    uint32_t t_first;
    if (whole) {
      t_first = nt > 0 ? steps % static_cast<uint32_t>(nt) : 0u;
    } else if (gr.kt == 0) {
      t_first = static_cast<uint32_t>(nt - take);
    } else {
      const int64_t start = at - gr.kt;
      const int64_t cut = p16_share(tiles, p16_holder(tiles, start, takers) + 1, takers);
      t_first = static_cast<uint32_t>(gr.kt - static_cast<int>(cut - start));
    }
    steps += static_cast<uint32_t>(count);
    const int t0 = __builtin_amdgcn_readfirstlane(static_cast<int>(t_first));
    auto after = [&](int t) { return t + 1 == nt ? 0 : t + 1; };
    int buf = 0;
    // The last unit's reads of both buffers are done (its stores may be on
    // their way).
    lds_barrier();
    // Page numbers are read a tile before their loads.
    int32_t entry = 0;
    if (count > 0) {
      entry = kPage16 ? ld_ro(table, page(t0)) : 0;
      load(t0, 0, entry);
      entry = kPage16 ? ld_ro(table, page(after(t0))) : 0;
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
    // A wave without rows only loads, and leaves its SIMD to the others: 32 rows
    // of 64 requests against 1,500 keys 82.6 -> 79.0 us, 20 ragged requests 34.6
    // -> 33.8 (16 short prompts at D = 64 41.1 -> 39.6). At D = 256 there is no
    // other wave, and the registers' spills grow (708 -> 733).
    if constexpr (D != 256) {
      if (32 * wave >= rows) {
        for (int i = 0, next = after(t0); i < count; ++i, next = after(next), buf ^= 1) {
          wait_vmcnt<0>();
          __syncthreads();
          if (i + 1 < count) {
            load(next, buf ^ 1, entry);
            entry = kPage16 ? ld_ro(table, page(after(next))) : 0;
          }
        }
        continue;
      }
    }
    for (int i = 0, t = t0, next = after(t0); i < count;
         ++i, t = next, next = after(next), buf ^= 1) {
      wait_vmcnt<0>();
      __syncthreads();  // tile t is in LDS, and nobody reads tile t - 1 any more
      if (i + 1 < count) load(next, buf ^ 1, entry);
      const char* kt = lds + buf * W::kBuf;
      const char* vt = kt + 2 * W::kBuf;

      // Scores: K operands four products ahead.
      f32x16 s[2];
      u32x4 kf[2][4];
      auto read_k = [&](int n) {
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
      auto read_v = [&](int i) {
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
      // The softmax goes before the scores, and these before the PV products, of
      // the SIMD's other waves, so that they run beside each other (4 x 2,048 rows
      // against 4,096 keys: 586 us with the softmax before both, 576 so; on
      // another card 556 without, 540 with the first, 541 with the products first).
      __builtin_amdgcn_s_setprio(2);
      read_v(0);
      // The page number for the next tile but one, on its way during the
      // softmax and waited for behind it: counted with LDS reads, which it
      // would otherwise make wait for all.
      if constexpr (kPage16) {
        __builtin_amdgcn_sched_barrier(0);
        entry = ld_ro(table, page(after(next)));
      }
      if (kKT * t + kKT > len) {
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const int key = kKT * t + 32 * b + 8 * (i >> 2) + 4 * h + (i & 3);
            s[b][i] = key < len ? s[b][i] : kNegInf;
          }
      }
      // The first maximum is the compiler's, which waits for the last product
      // (and so for all before it); it does not wait for an asm operand.
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
        // In place: otherwise the branch costs a copy of O in every tile. The
        // compiler does not see that the first product needs a wait after the
        // exp2; O's own products were issued before the scores'.
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
      const float shift = (m == kNegInf ? 0.0f : m) - kBias;
      u32x4 pf[4];
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int i = 0; i < 16; i += 2) {
          const float x0 = __builtin_amdgcn_exp2f(s[b][i] * p.scale_log2 - shift);
          const float x1 = __builtin_amdgcn_exp2f(s[b][i + 1] * p.scale_log2 - shift);
          const uint32_t w = pack16<kF16>(x0, x1);
          l = add_pair<kF16>(w, l);
          pf[2 * b + (i >> 3)][(i & 7) >> 1] = w;
        }
      if constexpr (kPage16) asm volatile("" ::"s"(entry));
      __builtin_amdgcn_s_setprio(0);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        __builtin_amdgcn_sched_barrier(0);
        if (i < 3) read_v(i + 1);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int j = 0; j < W::kO; ++j) o[j] = mfma32<kF16>(vf[i & 1][j], pf[i], o[j]);
      }
      __builtin_amdgcn_s_setprio(1);
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
      // A row without keys is 0; one whose scores are all -inf is 0 / 0, NaN.
      const float inv = 1.0f / sum;
      char* dst = p.out + token * p.s_out_tok + head * p.s_out_head + 8 * h;
#pragma unroll
      for (int j = 0; j < W::kO; ++j)
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          const u32x2 y = {pack16<kF16>(o[j][4 * b] * inv, o[j][4 * b + 1] * inv),
                           pack16<kF16>(o[j][4 * b + 2] * inv, o[j][4 * b + 3] * inv)};
          *reinterpret_cast<u32x2*>(dst + 64 * j + 16 * b) = len == 0 ? (u32x2){0u, 0u} : y;
        }
    }
  }
  if (!noted && threadIdx.x == 0) p16_note_none<D>(p, wg);
}

template <int D>
hipError_t wide_kernel(const P16Params& p, bool f16, bool page16, hipStream_t stream) {
  const dim3 grid(static_cast<unsigned>(p.num_wg)), block(64 * kP16Waves);
  if (f16 && page16) hipLaunchKernelGGL((p16_wide<D, true, true>), grid, block, 0, stream, p);
  else if (f16) hipLaunchKernelGGL((p16_wide<D, true, false>), grid, block, 0, stream, p);
  else if (page16) hipLaunchKernelGGL((p16_wide<D, false, true>), grid, block, 0, stream, p);
  else hipLaunchKernelGGL((p16_wide<D, false, false>), grid, block, 0, stream, p);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_p16_wide_kernel(const P16Params& p, bool f16, bool page16, int head_size,
                                  hipStream_t stream) {
  note_kernel("p16_wide");
  switch (head_size) {
    case 64: return wide_kernel<64>(p, f16, page16, stream);
    case 256: return wide_kernel<256>(p, f16, page16, stream);
    default: return wide_kernel<128>(p, f16, page16, stream);
  }
}

}  // namespace pa
