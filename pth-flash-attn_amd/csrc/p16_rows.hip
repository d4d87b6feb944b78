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
// 22 significant bits): the second product costs matrix time that this kernel
// has to spare, being bound by the cache's bytes. A masked key takes the
// address of a visible one and the weight 0, so nothing behind a request's
// last key, or in another's page, can reach a sum, whatever it holds.

#include "attn_device.h"
#include "p16.h"

namespace pa {
namespace {

template <int D>
struct RowsDim {
  static constexpr int kQ = D / 32;                  // QK products per 16 keys
  static constexpr int kCols = D < 128 ? D / 16 : 8; // columns per V load
  static constexpr int kPieces = D / (16 * kCols);   // V loads per key row
  static constexpr int kO = D / 16;                  // PV products per chunk
  static constexpr int kPerSimd = D == 64 ? 4 : D == 128 ? 3 : 1;
};

template <int kCols>
struct VRun;
template <>
struct VRun<4> { typedef u32x2 type; };
template <>
struct VRun<8> { typedef u32x4 type; };

template <bool kF16>
__device__ __forceinline__ f32x4 mfma16(u32x4 a, u32x4 b, f32x4 c) {
  if constexpr (kF16)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a),
                                                  __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a),
                                                   __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

// Two fp32 -> two 16-bit values, to nearest even.
template <bool kF16>
__device__ __forceinline__ uint32_t pack16(float a, float b) {
  if constexpr (kF16)
    return __builtin_bit_cast(uint32_t,
                              __builtin_convertvector((f32x2){a, b}, f16x2));
  else
    return __builtin_bit_cast(uint32_t, pack_bf16(a, b));
}
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

// The cache rows of 16-key blocks as a lane addresses them: with pages of a
// multiple of 16 slots, one page per block, its number read on the scalar
// unit; otherwise one page per key.
template <bool kPage16>
struct Walker {
  const P16Params& p;
  const int32_t* table;  // the request's row of the block table
  int32_t lo, len;       // visible keys
  int64_t head;

  __device__ __forceinline__ int32_t page(int32_t index) const {
    const int32_t id = ld_ro(table, index);
    return static_cast<uint32_t>(id) < static_cast<uint32_t>(p.num_blocks) ? id : 0;
  }
  // The block that stands for the 16 keys from k0 on: itself, or the last one.
  __device__ __forceinline__ int32_t block(int32_t k0) const { return min(k0, (len - 1) & ~15); }
  __device__ __forceinline__ int32_t block_page(int32_t kb) const {
    return kPage16 ? page(static_cast<int32_t>(p.bs_div.div(static_cast<uint32_t>(kb)))) : 0;
  }
  // Address of key kb + i (brought into the visible keys) of stream s; id:
  // the block's page.
  __device__ __forceinline__ const char* row(const CacheStream& s, int32_t kb, int32_t id,
                                             int32_t i) const {
    const int32_t at = min(max(i, lo - kb), len - 1 - kb);
    if constexpr (kPage16) {
      const int32_t first = kb - static_cast<int32_t>(p.bs_div.div(static_cast<uint32_t>(kb)) * p.bs_div.d);
      const char* b = s.base + static_cast<int64_t>(id) * s.s_block +
                      static_cast<int64_t>(first) * s.s_slot + head * s.s_head;
      return b + __umul24(static_cast<uint32_t>(at), static_cast<uint32_t>(s.s_slot));
    } else {
      const uint32_t key = static_cast<uint32_t>(kb + at);
      const uint32_t pg = p.bs_div.div(key);
      int32_t n = table[pg];
      n = static_cast<uint32_t>(n) < static_cast<uint32_t>(p.num_blocks) ? n : 0;
      return s.base + static_cast<int64_t>(n) * s.s_block +
             static_cast<int64_t>(key - pg * p.bs_div.d) * s.s_slot + head * s.s_head;
    }
  }
};

template <int D, bool kF16, bool kPage16>
__global__ __launch_bounds__(64 * kP16Waves, RowsDim<D>::kPerSimd) void p16_rows(
    const P16Params p) {
  using R = RowsDim<D>;
  using V = typename VRun<R::kCols>::type;
  constexpr int kBM = kP16RowsRows, kKT = kP16RowsKeys, kStride = D + 4;
  __shared__ float s_m[kP16Waves][kBM], s_l[kP16Waves][kBM], s_tot[kBM];
  __shared__ float s_o[kP16Waves][kBM * kStride];

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r16 = lane & 15, g = lane >> 4;
  P16Cursor cur;
  const int64_t tiles = p16_begin<kBM, kKT>(p, cur, lane);
  const int takers = p16_takers(p, tiles);
  if (static_cast<int>(blockIdx.x) >= takers) return;
  int64_t at = p16_share(tiles, blockIdx.x, takers);
  const int64_t end = p16_share(tiles, blockIdx.x + 1, takers);
  bool first = true;

  while (at < end) {
    const P16Unit u = p16_locate<kBM, kKT>(p, cur, at, lane);
    const int take = static_cast<int>(min(static_cast<int64_t>(u.req.n_kt - u.kt), end - at));
    const bool whole = take == u.req.n_kt;
    const int slot = 2 * static_cast<int>(blockIdx.x) + (u.kt == 0 ? 1 : 0);
    at += take;
    const int rows = min(kBM, u.req.rows - u.rt * kBM);

    // Q: 16 bytes per product, zeros in rows that the unit lacks.
    u32x4 q[R::kQ];
    {
      int64_t token, head;
      p16_row<kBM>(p, u, min(r16, rows - 1), token, head);
      const char* src = p.q + token * p.s_q_tok + head * p.s_q_head + 16 * g;
#pragma unroll
      for (int j = 0; j < R::kQ; ++j) {
        q[j] = *reinterpret_cast<const u32x4*>(src + 64 * j);
        if (r16 >= rows) q[j] = (u32x4){0u, 0u, 0u, 0u};
      }
    }

    float m = kNegInf, l = 0.0f;
    f32x4 o[R::kO];
#pragma unroll
    for (int j = 0; j < R::kO; ++j) o[j] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};

    Walker<kPage16> w{p, p.block_table + static_cast<int64_t>(u.r) * p.bt_stride, u.req.lo,
                      u.req.len, u.head};
    const int k_end = min(u.req.base + (u.kt + take) * kKT, u.req.len);
    int k0 = u.req.base + u.kt * kKT + 32 * wave;

    u32x4 kf[2][R::kQ];
    V vf[8][R::kPieces];
    auto load_k = [&](int kk, const int32_t (&id)[2]) {
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        const char* src = w.row(p.k, w.block(kk + 16 * b), id[b], r16) + 16 * g;
#pragma unroll
        for (int j = 0; j < R::kQ; ++j) kf[b][j] = *reinterpret_cast<const u32x4*>(src + 64 * j);
      }
    };
    auto load_v = [&](int kk, const int32_t (&id)[2]) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const char* src = w.row(p.v, w.block(kk + 16 * (e >> 2)), id[e >> 2], 4 * g + (e & 3)) +
                          2 * R::kCols * r16;
#pragma unroll
        for (int c = 0; c < R::kPieces; ++c) vf[e][c] = *reinterpret_cast<const V*>(src + 256 * c);
      }
    };
    if (k0 < k_end) {
      int32_t id[2] = {w.block_page(w.block(k0)), w.block_page(w.block(k0 + 16))};
      load_k(k0, id);
      load_v(k0, id);
      for (;;) {
        const int next = k0 + kKT;
        const bool more = next < k_end;
        if (more) {
          id[0] = w.block_page(w.block(next));
          id[1] = w.block_page(w.block(next + 16));
        }
        f32x4 s[2];
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          s[b] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
          for (int j = 0; j < R::kQ; ++j) s[b] = mfma16<kF16>(kf[b][j], q[j], s[b]);
        }
        if (more) load_k(next, id);
        float t[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) t[e] = s[e >> 2][e & 3] * p.scale_log2;
        if (k0 < u.req.lo || k0 + 32 > u.req.len) {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const int key = k0 + 16 * (e >> 2) + 4 * g + (e & 3);
            t[e] = key >= u.req.lo && key < u.req.len ? t[e] : kNegInf;
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
          x[e] = __builtin_amdgcn_exp2f(t[e] - ref);
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
        if (!more) break;
        load_v(next, id);
        k0 = next;
      }
    }

    // Join the four waves: all of them rescaled to the work-group's maximum.
    l = xor_sum(l);
    if (!first) __syncthreads();  // the last unit's sums have been read
    first = false;
    if (g == 0) {
      s_m[wave][r16] = m;
      s_l[wave][r16] = l;
    }
    __syncthreads();
    float top = s_m[0][r16];
#pragma unroll
    for (int i = 1; i < kP16Waves; ++i) top = fmaxf(top, s_m[i][r16]);
    const float ref = top == kNegInf ? 0.0f : top;
    const float f = __builtin_amdgcn_exp2f(m - ref);
    if (threadIdx.x < kBM) {
      float sum = 0.0f;
#pragma unroll
      for (int i = 0; i < kP16Waves; ++i)
        sum += s_l[i][r16] * __builtin_amdgcn_exp2f(s_m[i][r16] - ref);
      s_tot[r16] = sum;
      if (!whole && r16 < rows) {
        float* ml = p16_slot_ml<kBM, D>(p, slot) + 2 * r16;
        ml[0] = top;
        ml[1] = sum;
      }
    }
    if (r16 < rows) {
      // Lane's output column of product (c, j), register i: 16 kCols c + kCols (4 g + i) + j.
#pragma unroll
      for (int c = 0; c < R::kPieces; ++c)
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 0; j < R::kCols; j += 4) {
            f32x4 x;
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] = o[c * R::kCols + j + e][i] * f;
            *reinterpret_cast<f32x4*>(&s_o[wave][r16 * kStride + 16 * R::kCols * c +
                                                 R::kCols * (4 * g + i) + j]) = x;
          }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < rows * (D / 4); i += 64 * kP16Waves) {
      const int row = i / (D / 4), col = 4 * (i % (D / 4));
      f32x4 x = *reinterpret_cast<const f32x4*>(&s_o[0][row * kStride + col]);
#pragma unroll
      for (int v = 1; v < kP16Waves; ++v)
        x += *reinterpret_cast<const f32x4*>(&s_o[v][row * kStride + col]);
      if (!whole) {
        *reinterpret_cast<f32x4*>(p16_slot_o<kBM, D>(p, slot) + row * D + col) = x;
        continue;
      }
      // A row without keys is 0; one whose scores are all -inf is 0 / 0, NaN.
      const float inv = 1.0f / s_tot[row];
      const bool none = u.req.len == 0;
      int64_t token, head;
      p16_row<kBM>(p, u, row, token, head);
      u32x2 y;
#pragma unroll
      for (int e = 0; e < 2; ++e)
        y[e] = none ? 0u : pack16<kF16>(x[2 * e] * inv, x[2 * e + 1] * inv);
      *reinterpret_cast<u32x2*>(p.out + token * p.s_out_tok + head * p.s_out_head + 2 * col) = y;
    }
  }
}

// Joins the units that the partition cut (p16.h): work-group (w, y) the unit
// that begins in w and goes on in w + 1, rows y, y + gridDim.y and so on. Per
// row M = max m_s, L = sum l_s 2^(m_s - M), out = sum o_s 2^(m_s - M) / L, the
// slots in a fixed order.
template <int D, bool kF16, int kBM, int kKT>
__global__ __launch_bounds__(256) void p16_combine(const P16Params p) {
  constexpr int kVec = D / 4, kGroups = 256 / kVec;
  __shared__ float s_w[256];
  __shared__ float s_red[4];
  __shared__ f32x4 s_x[kGroups][kVec];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, tid = threadIdx.x;
  const int wg = blockIdx.x;
  P16Cursor cur;
  const int64_t tiles = p16_begin<kBM, kKT>(p, cur, lane);
  const int takers = p16_takers(p, tiles);
  if (wg + 1 >= takers) return;  // the last one's units end in it
  const int64_t begin = p16_share(tiles, wg, takers);
  const int64_t end = p16_share(tiles, wg + 1, takers);
  const P16Unit u = p16_locate<kBM, kKT>(p, cur, end - 1, lane);
  const int64_t u0 = end - 1 - u.kt, u1 = u0 + u.req.n_kt;
  if (u0 < begin || u1 <= end) return;  // begins before wg, or ends in it
  const int slots = p16_holder(tiles, u1 - 1, takers) - wg + 1;
  const int rows = min(kBM, u.req.rows - u.rt * kBM);
  const int col = tid % kVec, grp = tid / kVec;
  auto slot_of = [&](int s) { return s == 0 ? 2 * wg + 1 : 2 * (wg + s); };

  for (int row = blockIdx.y; row < rows; row += gridDim.y) {
    float top = kNegInf;
    for (int s = tid; s < slots; s += 256)
      top = fmaxf(top, p16_slot_ml<kBM, D>(p, slot_of(s))[2 * row]);
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) top = fmaxf(top, __shfl_xor(top, d));
    __syncthreads();  // the last row's sums have been read
    if (lane == 0) s_red[wave] = top;
    __syncthreads();
    top = fmaxf(fmaxf(s_red[0], s_red[1]), fmaxf(s_red[2], s_red[3]));
    const float ref = top == kNegInf ? 0.0f : top;
    f32x4 x = {0.0f, 0.0f, 0.0f, 0.0f};
    float sum = 0.0f;
    for (int s0 = 0; s0 < slots; s0 += 256) {
      const int n = min(256, slots - s0);
      __syncthreads();
      float part = 0.0f;
      if (tid < n) {
        const float* ml = p16_slot_ml<kBM, D>(p, slot_of(s0 + tid)) + 2 * row;
        s_w[tid] = __builtin_amdgcn_exp2f(ml[0] - ref);
        part = ml[1] * s_w[tid];
      }
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) part += __shfl_xor(part, d);
      if (lane == 0) s_red[wave] = part;
      __syncthreads();
      sum += (s_red[0] + s_red[1]) + (s_red[2] + s_red[3]);
      for (int s = grp; s < n; s += kGroups)
        x += s_w[s] * *reinterpret_cast<const f32x4*>(p16_slot_o<kBM, D>(p, slot_of(s0 + s)) +
                                                      row * D + 4 * col);
    }
    s_x[grp][col] = x;
    __syncthreads();
    if (grp == 0) {
#pragma unroll
      for (int i = 1; i < kGroups; ++i) x += s_x[i][col];
      const float inv = 1.0f / sum;
      int64_t token, head;
      p16_row<kBM>(p, u, row, token, head);
      const u32x2 y = {pack16<kF16>(x[0] * inv, x[1] * inv), pack16<kF16>(x[2] * inv, x[3] * inv)};
      *reinterpret_cast<u32x2*>(p.out + token * p.s_out_tok + head * p.s_out_head + 8 * col) = y;
    }
  }
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

template <int D>
hipError_t combine_kernel(const P16Params& p, bool f16, bool wide, hipStream_t stream) {
  const int most = wide ? kP16WideRows : min(kP16RowsRows, p.group * (p.qsl ? 16 : 1));
  const dim3 grid(static_cast<unsigned>(p.num_wg), static_cast<unsigned>(min(most, 16))), block(256);
  if (wide) {
    if (f16)
      hipLaunchKernelGGL((p16_combine<D, true, kP16WideRows, kP16WideKeys>), grid, block, 0, stream, p);
    else
      hipLaunchKernelGGL((p16_combine<D, false, kP16WideRows, kP16WideKeys>), grid, block, 0, stream, p);
  } else {
    if (f16)
      hipLaunchKernelGGL((p16_combine<D, true, kP16RowsRows, kP16RowsKeys>), grid, block, 0, stream, p);
    else
      hipLaunchKernelGGL((p16_combine<D, false, kP16RowsRows, kP16RowsKeys>), grid, block, 0, stream, p);
  }
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

hipError_t launch_p16_combine_kernel(const P16Params& p, bool f16, bool wide, int head_size,
                                     hipStream_t stream) {
  switch (head_size) {
    case 64: return combine_kernel<64>(p, f16, wide, stream);
    case 256: return combine_kernel<256>(p, f16, wide, stream);
    default: return combine_kernel<128>(p, f16, wide, stream);
  }
}

}  // namespace pa
