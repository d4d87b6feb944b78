// torch_checks.h -- what the torch ops of torch_op_p16.cpp and torch_op_fp8.cpp
// share: checks of tensors (strides, memory that two of them share), the
// device and its stream, and the C structs' fields.

#pragma once

#include <ATen/core/Tensor.h>
#include <ATen/hip/impl/HIPGuardImplMasqueradingAsCUDA.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <hip/hip_runtime.h>
#include <torch/library.h>

#include <algorithm>
#include <climits>
#include <cmath>
#include <cstdint>
#include <cstring>
#include <initializer_list>
#include <utility>

#include "attn_internal.h"

namespace {

using at::Tensor;
using c10::ScalarType;

#define OP_CHECK(cond, ...) TORCH_CHECK((cond), op, ": ", __VA_ARGS__)

bool is16(const Tensor& t) {
  return t.scalar_type() == ScalarType::BFloat16 || t.scalar_type() == ScalarType::Half;
}
int64_t byte_stride(const Tensor& t, int64_t dim) {
  return t.stride(dim) * static_cast<int64_t>(t.element_size());
}
bool fits32(int64_t x) { return x <= INT32_MAX; }

// Bytes from the first element to one past the last; -1 for negative strides
// or more than int64 holds.
int64_t extent_bytes(const Tensor& t) {
  int64_t total = 1, term = 0;
  if (t.numel() == 0) return 0;
  for (int64_t i = 0; i < t.dim(); ++i) {
    if (t.stride(i) < 0 || __builtin_mul_overflow(t.size(i) - 1, t.stride(i), &term) ||
        __builtin_add_overflow(total, term, &total))
      return -1;
  }
  return __builtin_mul_overflow(total, static_cast<int64_t>(t.element_size()), &total) ? -1 : total;
}
// The bytes that a tensor spans.
struct Span {
  uintptr_t begin, end;
};
Span span_of(const char* op, const Tensor& t) {
  const int64_t n = extent_bytes(t);
  OP_CHECK(n >= 0, "negative strides, or a byte extent that overflows int64");
  const auto p = n > 0 ? reinterpret_cast<uintptr_t>(t.data_ptr()) : 0;
  return {p, p + static_cast<uintptr_t>(n)};
}
// Whether two elements may share memory: a dimension steps within the reach of
// those of smaller strides.
bool overlaps_itself(const Tensor& t) {
  const int64_t n = t.dim();
  int64_t order[4] = {0, 1, 2, 3};
  std::sort(order, order + n, [&](int64_t a, int64_t b) { return t.stride(a) < t.stride(b); });
  int64_t reach = 1;
  for (int64_t i = 0; i < n; ++i) {
    const int64_t d = order[i];
    if (t.size(d) <= 1) continue;
    if (t.stride(d) < reach) return true;
    reach = t.stride(d) * (t.size(d) - 1) + reach;
  }
  return false;
}
bool overlap(const Span& a, const Span& b) { return a.begin < b.end && b.begin < a.end; }

bool same_view(const Tensor& a, const Tensor& b) {
  if (a.data_ptr() != b.data_ptr() || a.sizes() != b.sizes()) return false;
  for (int64_t i = 0; i < a.dim(); ++i)
    if (a.size(i) > 1 && a.stride(i) != b.stride(i)) return false;
  return true;
}
// Whether two tensors of one type, at most 4-D, share an element: whether
// sum n_i s_i is the distance between their first elements for some n_i in
// [lo_i, hi_i], s_i the strides of both (b's counted backwards), from the
// largest on. What the smaller ones reach leaves one or two n_i of each where
// the strides nest; views that would take more than kMost steps count as
// sharing one.
class SharedElement {
 public:
  static bool of(const Tensor& a, const Tensor& b) {
    SharedElement x;
    if (a.numel() == 0 || b.numel() == 0) return false;
    for (int64_t i = 0; i < a.dim(); ++i) x.add(a.stride(i), 0, a.size(i) - 1);
    for (int64_t i = 0; i < b.dim(); ++i) x.add(b.stride(i), 1 - b.size(i), 0);
    std::sort(x.terms_, x.terms_ + x.n_,
              [](const Term& p, const Term& q) { return p.stride > q.stride; });
    for (int64_t i = x.n_; i-- > 0;) {
      x.lo_[i] = x.lo_[i + 1] + x.terms_[i].lo * x.terms_[i].stride;
      x.hi_[i] = x.hi_[i + 1] + x.terms_[i].hi * x.terms_[i].stride;
    }
    const int64_t apart = reinterpret_cast<intptr_t>(b.data_ptr()) -
                          reinterpret_cast<intptr_t>(a.data_ptr());
    const int64_t size = static_cast<int64_t>(a.element_size());
    return apart % size != 0 || x.reaches(0, apart / size);
  }

 private:
  static constexpr int kMost = 1 << 16;
  struct Term {
    int64_t stride, lo, hi;
  };
  Term terms_[8];
  int64_t n_ = 0, lo_[9] = {}, hi_[9] = {};
  int steps_ = 0;

  void add(int64_t stride, int64_t lo, int64_t hi) {
    if (stride == 0 || lo == hi) return;
    for (int64_t i = 0; i < n_; ++i) {
      if (terms_[i].stride != stride) continue;
      terms_[i].lo += lo;
      terms_[i].hi += hi;
      return;
    }
    terms_[n_++] = {stride, lo, hi};
  }
  // Whether the terms from i on can sum to x.
  bool reaches(int64_t i, int64_t x) {
    if (x < lo_[i] || x > hi_[i]) return false;
    if (i == n_) return true;
    if (++steps_ > kMost) return true;
    const Term& t = terms_[i];
    const auto floor = [](int64_t a, int64_t b) { return a / b - (a % b < 0); };
    const int64_t from = std::max(t.lo, -floor(hi_[i + 1] - x, t.stride));
    const int64_t to = std::min(t.hi, floor(x - lo_[i + 1], t.stride));
    for (int64_t n = from; n <= to; ++n)
      if (reaches(i + 1, x - n * t.stride)) return true;
    return false;
  }
};

// The kernels are built for gfx950; a device's name does not change.
void check_device_arch(const char* op, const Tensor& t) {
  constexpr int kMost = 64;
  static bool known[kMost] = {};
  const int dev = t.get_device();
  if (dev < kMost && known[dev]) return;
  hipDeviceProp_t prop;
  const hipError_t err = hipGetDeviceProperties(&prop, dev);
  OP_CHECK(err == hipSuccess, "cannot query the device properties: ", hipGetErrorString(err));
  OP_CHECK(std::strncmp(prop.gcnArchName, "gfx950", 6) == 0,
           "needs a gfx950 (MI355X) device, device is ", prop.gcnArchName);
  if (dev < kMost) known[dev] = true;
}
void check_on_gpu(const char* op, const Tensor& t) {
  OP_CHECK(t.is_cuda(),
           "arguments are valid, but the op computes on CUDA tensors only (the CPU "
           "registration exists to test the argument checks)");
  check_device_arch(op, t);
}
hipStream_t stream_of_device(const Tensor& t) {
  return c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(t.get_device()).stream();
}
PthAttnStream stream_of(const Tensor& t) {
  PthAttnStream s{};
  s.data = t.data_ptr();
  s.stride_block = byte_stride(t, 0);
  s.stride_slot = byte_stride(t, 1);
  s.stride_head = byte_stride(t, 2);
  return s;
}
int32_t dtype_code(ScalarType t) {
  return t == ScalarType::Float ? PTH_ATTN_F32
         : t == ScalarType::Half ? PTH_ATTN_F16
                                 : PTH_ATTN_BF16;
}

}  // namespace
