// rotary.hip -- rotary positions: each pair (a, b) of a head's first rot_dim
// columns turns by its token's position times the pair's frequency,
//   (a, b) -> s (a cos - b sin, b cos + a sin).
//
// Angles. A frequency is held in turns per position as a 64-bit fraction, so
// that the 64-bit product with the position, wrapped, is the angle's place in
// the circle: exact at every position, where a 32-bit product loses an angle at
// position 10^6 to 0.06 radians, and without a table, whose rows would have to
// be read and reach to the last position. Its top 32 bits are split into a
// quadrant and the remainder within an eighth of a turn. In radians that is a sum
// a + e of two 32-bit values, and sine and cosine are a and 1 - a^2 / 2 with all the
// rest of their Taylor sums (to x^11 and x^10, (pi / 4)^12 / 12! = 1.1e-10 left)
// added at once, so that each is within 4.7e-8 of the exact value (rms 1.15e-8 and
// 1.72e-8, as 32 bits can be: 1.13e-8 and 1.72e-8).
//
// A work-group takes a few tokens: its threads first make the cosines and sines
// of all their pairs, one each, in LDS, for all heads; then each moves 16 bytes
// of pairs side by side, or of pairs' first and of their second members. Rows
// that are not on 16-byte addresses, or a rot_dim that does not divide so, take
// steps of 4 bytes or of one value. Stores go past the caches: the outputs of a
// large call do not fit them.
//
// Bound: its bytes (16,384 tokens, 32 + 8 heads of 128, bf16, cold: 335 MB, 64.5 us, 5.2 TB/s);
// latency for a decode step (64 tokens 2.7 us).

#include <hip/hip_runtime.h>

#include <algorithm>
#include <climits>
#include <cmath>
#include <string>

#include "attn_device.h"
#include "fp8.h"

namespace pa {
namespace {

struct RotaryParams {
  const char *q, *k;
  char *q_out, *k_out;
  int64_t s_q_tok, s_q_head, s_k_tok, s_k_head;
  int64_t s_qo_tok, s_qo_head, s_ko_tok, s_ko_head;
  const int64_t* positions;
  const int64_t* turns;
  Div32 half_div, row_div, heads_div;  // pairs of a head; items of a head; heads
  int32_t num_tokens, num_q_heads, heads;
  int32_t half;       // pairs
  int32_t row_items;  // of a head: runs of pairs, then runs of the rest
  int32_t pair_items;
  int32_t tokens;  // of a work-group
  int32_t sign;
  float scale;
};

constexpr int kRotThreads = 256;
constexpr int kRotPairs = 1024;  // cosines and sines that a work-group holds

// Sine and cosine of x 2 pi / 2^32.
__device__ __forceinline__ f32x2 sin_cos_turn(uint32_t x) {
#pragma clang fp contract(off)  // a, as it is rounded, is what e is the remainder of
  constexpr float kHi = 0x1.921fb6p-30f, kLo = -0x1.777a5cp-55f;  // 2 pi / 2^32, of two values
  const uint32_t q = (x + 0x20000000u) >> 30;
  const int32_t turn = static_cast<int32_t>(x - (q << 30));
  const int32_t top = (turn + 32) & ~63;  // 24 bits of it: exact, as what is left
  const float hi = static_cast<float>(top), lo = static_cast<float>(turn - top);
  const float a = hi * kHi;
  const float e = fmaf(lo, kHi, fmaf(hi, kLo, fmaf(hi, kHi, -a)));
  const float z = a * a;
  float s = fmaf(z, -2.5052108e-8f, 2.7557319e-6f);
  s = fmaf(z, s, -1.9841270e-4f);
  s = fmaf(z, s, 8.3333333e-3f);
  s = fmaf(z, s, -1.6666667e-1f);
  float c = fmaf(z, -2.7557319e-7f, 2.4801587e-5f);
  c = fmaf(z, c, -1.3888889e-3f);
  c = fmaf(z, c, 4.1666667e-2f);
  // 1 - z / 2 and what it was rounded by, z's own rounding, the angle's remainder.
  const float half = 0.5f * z, c0 = 1.0f - half, az = a * z;
  const float left =
      fmaf(-fmaf(az, s, a), e, fmaf(-0.5f, fmaf(a, a, -z), (1.0f - c0) - half));
  c = c0 + fmaf(z * z, c, left);
  s = a + fmaf(az, s, e * c);
  const float u = q & 1 ? c : s, v = q & 1 ? s : c;
  return (f32x2){q & 2 ? -u : u, (q + 1) & 2 ? -v : v};
}

// A run of kBytes of values of type T, as 32-bit ones.
template <class T, int kBytes>
struct Run {
  static constexpr int kN = kBytes / static_cast<int>(sizeof(T));
  typedef uint32_t Words __attribute__((ext_vector_type(kBytes / 4)));
  static __device__ __forceinline__ void load(const char* src, float (&x)[kN]) {
    T y[kN];
    const Words w = *reinterpret_cast<const Words*>(src);
    __builtin_memcpy(y, &w, kBytes);
#pragma unroll
    for (int i = 0; i < kN; ++i) x[i] = static_cast<float>(y[i]);
  }
  static __device__ __forceinline__ void store(char* dst, const float (&x)[kN]) {
    T y[kN];
#pragma unroll
    for (int i = 0; i < kN; ++i) y[i] = static_cast<T>(x[i]);
    Words w;
    __builtin_memcpy(&w, y, kBytes);
    __builtin_nontemporal_store(w, reinterpret_cast<Words*>(dst));
  }
};
template <class T>
struct Run<T, 2> {
  static constexpr int kN = 1;
  static __device__ __forceinline__ void load(const char* src, float (&x)[1]) {
    x[0] = static_cast<float>(*reinterpret_cast<const T*>(src));
  }
  static __device__ __forceinline__ void store(char* dst, const float (&x)[1]) {
    *reinterpret_cast<T*>(dst) = static_cast<T>(x[0]);
  }
};

template <class T, bool kInterleaved, int kBytes>
__global__ __launch_bounds__(kRotThreads) void rotary(const RotaryParams p) {
  using R = Run<T, kBytes>;
  __shared__ f32x2 s_turn[kRotPairs];
  const int t0 = static_cast<int>(blockIdx.x) * p.tokens;
  const int tokens = min(p.tokens, p.num_tokens - t0);
  for (int i = threadIdx.x; i < tokens * p.half; i += kRotThreads) {
    const uint32_t t = p.half_div.div(static_cast<uint32_t>(i));
    const uint64_t at = static_cast<uint64_t>(p.positions[t0 + static_cast<int>(t)]) *
                        static_cast<uint64_t>(p.turns[i - static_cast<int>(t) * p.half]);
    f32x2 x = sin_cos_turn(static_cast<uint32_t>((at + 0x80000000u) >> 32));
    s_turn[i] = (f32x2){x[0] * (p.sign < 0 ? -p.scale : p.scale), x[1] * p.scale};
  }
  __syncthreads();
  const int items = tokens * p.heads * p.row_items;
  const int step = static_cast<int>(gridDim.y) * kRotThreads;
  for (int i = static_cast<int>(blockIdx.y) * kRotThreads + static_cast<int>(threadIdx.x);
       i < items; i += step) {
    const int row = static_cast<int>(p.row_div.div(static_cast<uint32_t>(i)));
    const int c = i - row * p.row_items;
    const int t = static_cast<int>(p.heads_div.div(static_cast<uint32_t>(row)));
    int head = row - t * p.heads;
    const int64_t token = t0 + t;
    const bool is_q = head < p.num_q_heads;
    head -= is_q ? 0 : p.num_q_heads;
    const char* src = is_q ? p.q + token * p.s_q_tok + head * p.s_q_head
                           : p.k + token * p.s_k_tok + head * p.s_k_head;
    char* dst = is_q ? p.q_out + token * p.s_qo_tok + head * p.s_qo_head
                     : p.k_out + token * p.s_ko_tok + head * p.s_ko_head;
    const int64_t half_bytes = static_cast<int64_t>(p.half) * sizeof(T);
    if (c < p.pair_items) {
      if constexpr (kInterleaved && R::kN > 1) {  // a run of whole pairs
        const f32x2* turn = s_turn + t * p.half + c * (R::kN / 2);
        float x[R::kN];
        R::load(src + kBytes * c, x);
#pragma unroll
        for (int j = 0; j < R::kN; j += 2) {
          const f32x2 w = turn[j / 2];
          const float u = x[j], v = x[j + 1];
          x[j] = fmaf(u, w[1], -(v * w[0]));
          x[j + 1] = fmaf(v, w[1], u * w[0]);
        }
        R::store(dst + kBytes * c, x);
      } else {
        const f32x2* turn = s_turn + t * p.half + c * R::kN;
        const int64_t first = static_cast<int64_t>(kInterleaved ? 2 * kBytes : kBytes) * c;
        const int64_t second = first + (kInterleaved ? kBytes : half_bytes);
        float x[R::kN], y[R::kN];
        R::load(src + first, x);
        R::load(src + second, y);
#pragma unroll
        for (int j = 0; j < R::kN; ++j) {
          const f32x2 w = turn[j];
          const float u = x[j], v = y[j];
          x[j] = fmaf(u, w[1], -(v * w[0]));
          y[j] = fmaf(v, w[1], u * w[0]);
        }
        R::store(dst + first, x);
        R::store(dst + second, y);
      }
    } else if (src != dst) {  // behind the pairs; in place there is nothing to do
      const int64_t at = 2 * half_bytes + static_cast<int64_t>(kBytes) * (c - p.pair_items);
      float x[R::kN];
      R::load(src + at, x);
      R::store(dst + at, x);
    }
  }
}

template <class T, bool kInterleaved>
void rotary_of(const RotaryParams& p, int bytes, dim3 grid, hipStream_t stream) {
  if (bytes == 16) rotary<T, kInterleaved, 16><<<grid, kRotThreads, 0, stream>>>(p);
  else if (bytes == 4) rotary<T, kInterleaved, 4><<<grid, kRotThreads, 0, stream>>>(p);
  else if constexpr (sizeof(T) == 2) rotary<T, kInterleaved, 2><<<grid, kRotThreads, 0, stream>>>(p);
}
template <class T>
void rotary_as(const RotaryParams& p, bool interleaved, int bytes, dim3 grid, hipStream_t stream) {
  if (interleaved) rotary_of<T, true>(p, bytes, grid, stream);
  else rotary_of<T, false>(p, bytes, grid, stream);
}

}  // namespace

int32_t launch_rotary(const PthAttnRotaryArgs& a, hipStream_t stream) {
  clear_error();
  PA_REQUIRE(a.abi_version == PTH_ATTN_ABI_VERSION,
             "abi_version " + std::to_string(a.abi_version) + " != library ABI " +
                 std::to_string(PTH_ATTN_ABI_VERSION));
  PA_REQUIRE(a.struct_bytes == static_cast<int32_t>(sizeof(PthAttnRotaryArgs)),
             "struct_bytes " + std::to_string(a.struct_bytes) + " != sizeof(PthAttnRotaryArgs) " +
                 std::to_string(sizeof(PthAttnRotaryArgs)));
  PA_REQUIRE(a.dtype == PTH_ATTN_F32 || a.dtype == PTH_ATTN_F16 || a.dtype == PTH_ATTN_BF16,
             "dtype must be PTH_ATTN_F32, PTH_ATTN_F16 or PTH_ATTN_BF16");
  PA_REQUIRE(a.head_size >= 2 && a.head_size <= 1024, "head_size must be 2 .. 1024");
  PA_REQUIRE(a.rot_dim >= 2 && a.rot_dim % 2 == 0 && a.rot_dim <= a.head_size,
             "rot_dim must be even, 2 .. head_size");
  PA_REQUIRE(a.num_tokens >= 0 && a.num_q_heads >= 0 && a.num_kv_heads >= 0 &&
                 a.num_q_heads <= 1 << 16 && a.num_kv_heads <= 1 << 16,
             "num_tokens >= 0, num_q_heads and num_kv_heads 0 .. 65536");
  PA_REQUIRE(std::isfinite(a.scale), "scale must be finite");
  const int64_t heads = static_cast<int64_t>(a.num_q_heads) + a.num_kv_heads;
  if (a.num_tokens == 0 || heads == 0) return PTH_ATTN_OK;
  PA_REQUIRE((a.num_q_heads == 0 || (a.q && a.q_out)) && (a.num_kv_heads == 0 || (a.k && a.k_out)) &&
                 a.positions && a.turns,
             "q, k, q_out, k_out, positions and turns must be non-NULL");
  const int elt = a.dtype == PTH_ATTN_F32 ? 4 : 2;
  const int half = a.rot_dim / 2;
  // The widest step that every row's runs are aligned to and made of.
  const auto aligned = [&](int64_t n) {
    const auto on = [&](const void* p, int64_t tok, int64_t head, int64_t h) {
      return h == 0 || (reinterpret_cast<uintptr_t>(p) % n == 0 &&
                        used_stride(tok, a.num_tokens) % n == 0 && used_stride(head, h) % n == 0);
    };
    return on(a.q, a.q_stride_token, a.q_stride_head, a.num_q_heads) &&
           on(a.k, a.k_stride_token, a.k_stride_head, a.num_kv_heads) &&
           on(a.q_out, a.q_out_stride_token, a.q_out_stride_head, a.num_q_heads) &&
           on(a.k_out, a.k_out_stride_token, a.k_out_stride_head, a.num_kv_heads);
  };
  int bytes = elt;
  for (const int n : {16, 4}) {
    // A run holds n bytes: of whole pairs, or of its pairs' first members, and of their
    // second ones.
    if (n > elt && (a.interleaved ? 2 : 1) * half * elt % n == 0 && (a.head_size - a.rot_dim) * elt % n == 0 && aligned(n)) {
      bytes = n;
      break;
    }
  }
  PA_REQUIRE(aligned(elt), "q, k, q_out and k_out must be aligned to their element");
  RotaryParams p{};
  p.q = static_cast<const char*>(a.q);
  p.k = static_cast<const char*>(a.k);
  p.q_out = static_cast<char*>(a.q_out);
  p.k_out = static_cast<char*>(a.k_out);
  p.s_q_tok = a.q_stride_token;
  p.s_q_head = a.q_stride_head;
  p.s_k_tok = a.k_stride_token;
  p.s_k_head = a.k_stride_head;
  p.s_qo_tok = a.q_out_stride_token;
  p.s_qo_head = a.q_out_stride_head;
  p.s_ko_tok = a.k_out_stride_token;
  p.s_ko_head = a.k_out_stride_head;
  p.positions = a.positions;
  p.turns = a.turns;
  p.num_tokens = a.num_tokens;
  p.num_q_heads = a.num_q_heads;
  p.heads = static_cast<int32_t>(heads);
  p.half = half;
  p.pair_items = (a.interleaved && bytes > elt ? 2 : 1) * half * elt / bytes;
  p.row_items = p.pair_items + (a.head_size - a.rot_dim) * elt / bytes;
  p.half_div = Div32::make(static_cast<uint32_t>(half));
  p.row_div = Div32::make(static_cast<uint32_t>(p.row_items));
  p.heads_div = Div32::make(static_cast<uint32_t>(heads));
  p.sign = a.inverse ? -1 : 1;
  p.scale = a.scale;
  p.tokens = std::max(1, std::min(kRotPairs / half, a.num_tokens >= 4096 ? 4 : 1));
  const int64_t items = heads * p.row_items * p.tokens;
  PA_REQUIRE(items < INT32_MAX, "heads x head_size is too large");
  const int64_t groups = (int64_t{a.num_tokens} + p.tokens - 1) / p.tokens;
  PA_REQUIRE(groups <= kMostThreads / kRotThreads, "num_tokens needs more than 2^32 threads");
  const dim3 grid(static_cast<unsigned>(groups),
                  static_cast<unsigned>(a.num_tokens >= 1024
                                            ? 1
                                            : std::min<int64_t>((items + kRotThreads - 1) / kRotThreads, 8)));
  if (a.dtype == PTH_ATTN_F32) rotary_as<float>(p, a.interleaved, bytes, grid, stream);
  else if (a.dtype == PTH_ATTN_F16) rotary_as<_Float16>(p, a.interleaved, bytes, grid, stream);
  else rotary_as<__bf16>(p, a.interleaved, bytes, grid, stream);
  const hipError_t err = hipGetLastError();
  if (err != hipSuccess)
    return fail(PTH_ATTN_ECUDA, std::string("rotary launch: ") + hipGetErrorString(err));
  return PTH_ATTN_OK;
}

}  // namespace pa

extern "C" {

int32_t pth_attn_rotary_args_bytes(void) { return static_cast<int32_t>(sizeof(PthAttnRotaryArgs)); }

int32_t pth_attn_rotary(const PthAttnRotaryArgs* args, void* stream) {
  if (args == nullptr) return pa::fail(PTH_ATTN_EINVAL, "args is NULL");
  return pa::launch_rotary(*args, static_cast<hipStream_t>(stream));
}

}  // extern "C"
