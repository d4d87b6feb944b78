// p16_combine.hip -- joins the groups that the partition of p16.h cut:
// work-group (i, y) the rows y, y + gridDim.y ... of the group of note i. Per row
//   M = max m_s, L = sum l_s 2^(m_s - M), out = sum o_s 2^(m_s - M) / L,
// the slots s in an order that the sizes fix.
//
// A crew of D / 4 lanes reads a row, four columns a lane. With few slots, or
// twice as many rows, each crew joins a row by itself; otherwise they share one
// row's slots and join in LDS (64 rows of 17 slots, whole call of 8 requests to
// 6,000 states: 41.0 us alone, 46.4 shared).
//
// Bound: latency (a note, then slots that the launch before wrote). One request
// to 128k keys, 128 slots of 4 rows: 4.6 us; 64 requests to 32k keys 5.1. Of
// 128-row units it is their bytes: 4 long prompts, up to 68 MB of slots, 20 us.

#include "attn_device.h"
#include "p16.h"

namespace pa {
namespace {

template <int D, bool kF16, int kBM, int kThreads, class P>
__global__ __launch_bounds__(kThreads) void p16_combine(const P p) {
  constexpr int kVec = D / 4, kCrews = kThreads / kVec, kAhead = kThreads > 256 ? 8 : 4;
  __shared__ f32x4 s_o[kCrews][kVec];
  __shared__ float s_m[kCrews], s_l[kCrews];
  const int col = threadIdx.x % kVec, crew = threadIdx.x / kVec;
  if (p16_counted(p) && blockIdx.x >= p16_cut<D>(p, 0)->slots_wg) return;
  const P16Cut cut = *p16_cut<D>(p, p.notes > 0 ? 1 + blockIdx.x : blockIdx.x);
  const int slots = cut.slots_wg & ((1u << kP16CutShift) - 1);
  const int wg = cut.slots_wg >> kP16CutShift;
  if (slots == 0) return;
  P16Req x;
  x.n_rt = (cut.rows + kBM - 1) / kBM;
  const int first = cut.group * p.team;
  const int subs = min(p.team, p.num_kv_heads * x.n_rt - first);
  const int items = subs * p.slot_rows;  // rows of the group, as a slot holds them
  const bool alone = slots <= max(8, items / 2);
  const int step = alone ? 1 : kCrews;
  for (int i = alone ? crew + kCrews * static_cast<int>(blockIdx.y) : static_cast<int>(blockIdx.y);
       i < items; i += (alone ? kCrews : 1) * static_cast<int>(gridDim.y)) {
    const int sub = i / p.slot_rows, row = i - sub * p.slot_rows;
    const P16Unit u = p16_unit(x, first + sub);
    if (row >= cut.rows - u.rt * kBM) continue;
    float m = kNegInf, l = 0.0f;
    f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
    // Slots s, s + step ..., kAhead reads at a time.
    for (int s = alone ? 0 : crew; s < slots; s += kAhead * step) {
      f32x4 so[kAhead];
      f32x2 ml[kAhead];
#pragma unroll
      for (int a = 0; a < kAhead; ++a) {
        const int n = min(s + a * step, slots - 1);
        const int at = n == 0 ? 2 * wg + 1 : 2 * (wg + n);
        so[a] = *reinterpret_cast<const f32x4*>(p16_slot_o<D>(p, at, sub, row) + 4 * col);
        ml[a] = *reinterpret_cast<const f32x2*>(p16_slot_ml<D>(p, at, sub, row));
        if (s + a * step >= slots) {
          so[a] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
          ml[a] = (f32x2){kNegInf, 0.0f};
        }
      }
      float top = m;
#pragma unroll
      for (int a = 0; a < kAhead; ++a) top = fmaxf(top, ml[a][0]);
      const float ref = top == kNegInf ? 0.0f : top;
      const float f = __builtin_amdgcn_exp2f(m - ref);
      m = top;
      l *= f;
      o *= f;
#pragma unroll
      for (int a = 0; a < kAhead; ++a) {
        const float w = __builtin_amdgcn_exp2f(ml[a][0] - ref);
        l += w * ml[a][1];
        o += w * so[a];
      }
    }
    if (!alone) {  // the crews share the row
      __syncthreads();  // the last one has been read
      s_o[crew][col] = o;
      if (col == 0) {
        s_m[crew] = m;
        s_l[crew] = l;
      }
      __syncthreads();
      if (crew != 0) continue;
      float top = m;
#pragma unroll
      for (int v = 1; v < kCrews; ++v) top = fmaxf(top, s_m[v]);
      const float ref = top == kNegInf ? 0.0f : top;
      const float f = __builtin_amdgcn_exp2f(m - ref);
      l *= f;
      o *= f;
#pragma unroll 5
      for (int v = 1; v < kCrews; ++v) {
        const float w = __builtin_amdgcn_exp2f(s_m[v] - ref);
        l += w * s_l[v];
        o += w * s_o[v][col];
      }
    }
    const float inv = P::kF8 && l == 0.0f ? 0.0f : 1.0f / l;
    int64_t token, head;
    p16_row<kBM>(p, cut.q0, u, row, token, head);
    *reinterpret_cast<u32x2*>(p.out + token * p.s_out_tok + head * p.s_out_head + 8 * col) =
        (u32x2){pack16<kF16>(o[0] * inv, o[1] * inv), pack16<kF16>(o[2] * inv, o[3] * inv)};
  }
}

template <int D, bool kF16, class P>
void combine_of(const P& p, bool wide, dim3 grid, hipStream_t stream) {
  if (wide) p16_combine<D, kF16, kP16WideRows, 256><<<grid, 256, 0, stream>>>(p);
  else if (p.notes > 0) p16_combine<D, kF16, kP16RowsRows, 512><<<grid, 512, 0, stream>>>(p);
  else p16_combine<D, kF16, kP16RowsRows, 256><<<grid, 256, 0, stream>>>(p);
}
template <int D, class P>
void combine(const P& p, bool f16, bool wide, dim3 grid, hipStream_t stream) {
  if (f16) combine_of<D, true>(p, wide, grid, stream);
  else combine_of<D, false>(p, wide, grid, stream);
}
template <class P>
hipError_t launch_combine(const P& p, bool f16, bool wide, int head_size, int y,
                          hipStream_t stream) {
  const dim3 grid(static_cast<unsigned>(p.notes > 0 ? p.notes : p.num_wg),
                  static_cast<unsigned>(y));
  switch (head_size) {
    case 64: combine<64>(p, f16, wide, grid, stream); break;
    case 256: combine<256>(p, f16, wide, grid, stream); break;
    default: combine<128>(p, f16, wide, grid, stream);
  }
  return hipGetLastError();
}

}  // namespace

hipError_t launch_p16_combine_kernel(const P16Params& p, bool f16, bool wide, int head_size,
                                     int y, hipStream_t stream) {
  return launch_combine(p, f16, wide, head_size, y, stream);
}
hipError_t launch_f8_combine_kernel(const F8Params& p, bool f16, bool wide, int head_size, int y,
                                    hipStream_t stream) {
  return launch_combine(p, f16, wide, head_size, y, stream);
}

}  // namespace pa
