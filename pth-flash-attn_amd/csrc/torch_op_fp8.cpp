// torch_op_fp8.cpp -- the torch ops around a paged cache in 8-bit floating
// point with a scale for each block of 16 slots and KV head: rotary_embedding,
// reshape_and_cache_fp8, gather_cache_fp8 and paged_attn_fp8_fwd (no
// counterparts in the reference). As torch_op_p16.cpp: the CUDA key checks and
// launches, on the current stream of the tensors' device, allocating nothing
// and reading nothing back; the CPU key checks and raises. The fakes in
// ops8.py make the same metadata checks with the same messages.

#include "fp8.h"
#include "torch_checks.h"

#include <c10/util/Optional.h>

#include <optional>
#include <string>

namespace {

bool is_value(const Tensor& t) { return is16(t) || t.scalar_type() == ScalarType::Float; }

// ---- rotary positions -----------------------------------------------------

void rotary_embedding(const Tensor& q_out, const Tensor& k_out, const Tensor& q, const Tensor& k,
                      const Tensor& positions, const Tensor& turns, bool interleaved, double scale,
                      bool inverse) {
  const char* op = "rotary_embedding";
  OP_CHECK(q.dim() == 3 && k.dim() == 3, "q and k must be 3-D [T, heads, D]");
  const int64_t T = q.size(0), D = q.size(2);
  OP_CHECK(k.size(0) == T && k.size(2) == D, "q and k must have the same T and D");
  OP_CHECK(D >= 2 && D <= 1024, "head size must be 2 to 1024, got ", D);
  OP_CHECK(is_value(q) && k.scalar_type() == q.scalar_type(),
           "q and k must both be float32, bfloat16 or float16");
  OP_CHECK(q_out.sizes() == q.sizes() && q_out.scalar_type() == q.scalar_type() &&
               k_out.sizes() == k.sizes() && k_out.scalar_type() == k.scalar_type(),
           "q_out and k_out must have the shapes and dtype of q and k");
  for (const Tensor* t : {&q, &k, &q_out, &k_out})
    OP_CHECK(t->stride(2) == 1, "q, k, q_out and k_out must have stride 1 in their last dimension");
  OP_CHECK(positions.dim() == 1 && positions.size(0) == T &&
               positions.scalar_type() == ScalarType::Long && positions.is_contiguous(),
           "positions must be contiguous int64 [T]");
  OP_CHECK(turns.dim() == 1 && turns.scalar_type() == ScalarType::Long && turns.is_contiguous() &&
               turns.size(0) >= 1 && 2 * turns.size(0) <= D,
           "turns must be contiguous int64 [rot_dim / 2], rot_dim 2 to D");
  OP_CHECK(std::isfinite(scale), "scale must be finite, got ", scale);
  for (const Tensor* t : {&k, &q_out, &k_out, &positions, &turns})
    OP_CHECK(t->device() == q.device(), "all tensors must be on the device of q");
  OP_CHECK(!overlaps_itself(q_out) && !overlaps_itself(k_out),
           "q_out and k_out must not overlap themselves");
  const Tensor* outs[] = {&q_out, &k_out};
  const Tensor* ins[] = {&q, &k};
  OP_CHECK(!SharedElement::of(q_out, k_out), "q_out and k_out must share no memory");
  for (int i = 0; i < 2; ++i) {
    const Span s = span_of(op, *outs[i]);
    for (int j = 0; j < 2; ++j)
      OP_CHECK(!overlap(s, span_of(op, *ins[j])) ||
                   (i == j && same_view(*outs[i], *ins[j])) ||
                   !SharedElement::of(*outs[i], *ins[j]),
               "an output must be its input itself or share no memory with one");
    for (const Tensor* t : {&positions, &turns})
      OP_CHECK(!overlap(s, span_of(op, *t)), "an output must not overlap positions or turns");
  }
  OP_CHECK(fits32(T) && q.size(1) <= 65536 && k.size(1) <= 65536, "a size exceeds its limit");
  check_on_gpu(op, q);
  const c10::hip::HIPGuardMasqueradingAsCUDA guard(q.device());
  PthAttnRotaryArgs a{};
  a.abi_version = PTH_ATTN_ABI_VERSION;
  a.struct_bytes = static_cast<int32_t>(sizeof(PthAttnRotaryArgs));
  a.q = q.data_ptr();
  a.q_stride_token = byte_stride(q, 0);
  a.q_stride_head = byte_stride(q, 1);
  a.k = k.data_ptr();
  a.k_stride_token = byte_stride(k, 0);
  a.k_stride_head = byte_stride(k, 1);
  a.q_out = q_out.data_ptr();
  a.q_out_stride_token = byte_stride(q_out, 0);
  a.q_out_stride_head = byte_stride(q_out, 1);
  a.k_out = k_out.data_ptr();
  a.k_out_stride_token = byte_stride(k_out, 0);
  a.k_out_stride_head = byte_stride(k_out, 1);
  a.positions = static_cast<const int64_t*>(positions.data_ptr());
  a.turns = static_cast<const int64_t*>(turns.data_ptr());
  a.dtype = dtype_code(q.scalar_type());
  a.num_tokens = static_cast<int32_t>(T);
  a.num_q_heads = static_cast<int32_t>(q.size(1));
  a.num_kv_heads = static_cast<int32_t>(k.size(1));
  a.head_size = static_cast<int32_t>(D);
  a.rot_dim = static_cast<int32_t>(2 * turns.size(0));
  a.interleaved = interleaved ? 1 : 0;
  a.inverse = inverse ? 1 : 0;
  a.scale = static_cast<float>(scale);
  const int32_t rc = pa::launch_rotary(a, stream_of_device(q));
  OP_CHECK(rc == PTH_ATTN_OK, pa::last_error());
}

// ---- the cache ------------------------------------------------------------

void check_cache_f8(const char* op, const Tensor& k, const Tensor& v, const Tensor& ks,
                    const Tensor& vs, int64_t D) {
  OP_CHECK(k.dim() == 4 && v.dim() == 4 && k.sizes() == v.sizes() && k.size(3) == D,
           "k_cache and v_cache must be [num_blocks, block_size, Hkv, ", D, "]");
  OP_CHECK(D == 64 || D == 128 || D == 256, "head size must be 64, 128 or 256, got ", D);
  OP_CHECK(k.scalar_type() == ScalarType::Float8_e4m3fn &&
               v.scalar_type() == ScalarType::Float8_e4m3fn,
           "k_cache and v_cache must be float8_e4m3fn");
  OP_CHECK(k.size(0) >= 1 && k.size(1) >= 1 && k.size(2) >= 1,
           "k_cache and v_cache must not be empty");
  OP_CHECK(k.size(1) % pa::kF8Span == 0, "block_size must be a multiple of 16, got ", k.size(1));
  OP_CHECK(k.stride(3) == 1 && v.stride(3) == 1,
           "k_cache and v_cache must have stride 1 in their last dimension");
  for (const Tensor* t : {&ks, &vs})
    OP_CHECK(t->dim() == 3 && t->scalar_type() == ScalarType::Byte && t->is_contiguous() &&
                 t->size(0) == k.size(0) && t->size(1) == k.size(1) / pa::kF8Span &&
                 t->size(2) == k.size(2),
             "k_scale and v_scale must be contiguous uint8 [num_blocks, block_size / 16, Hkv]");
}
PthAttnCacheF8 cache_of(const Tensor& k, const Tensor& v, const Tensor& ks, const Tensor& vs) {
  PthAttnCacheF8 c{};
  c.k_cache = stream_of(k);
  c.v_cache = stream_of(v);
  c.k_scale = static_cast<uint8_t*>(ks.data_ptr());
  c.v_scale = static_cast<uint8_t*>(vs.data_ptr());
  c.num_blocks = static_cast<int32_t>(k.size(0));
  c.block_size = static_cast<int32_t>(k.size(1));
  c.num_kv_heads = static_cast<int32_t>(k.size(2));
  c.head_size = static_cast<int32_t>(k.size(3));
  return c;
}
bool cache_fits32(const Tensor& k) {
  return fits32(k.size(0)) && fits32(k.size(1)) && fits32(k.size(2));
}

void reshape_and_cache_fp8(const Tensor& key, const Tensor& value, const Tensor& k_cache,
                           const Tensor& v_cache, const Tensor& k_scale, const Tensor& v_scale,
                           const Tensor& slot_mapping) {
  const char* op = "reshape_and_cache_fp8";
  OP_CHECK(key.dim() == 3 && value.dim() == 3, "key and value must be 3-D [T, Hkv, D]");
  OP_CHECK(key.sizes() == value.sizes(), "key and value must have the same shape");
  const int64_t T = key.size(0);
  check_cache_f8(op, k_cache, v_cache, k_scale, v_scale, key.size(2));
  OP_CHECK(k_cache.size(2) == key.size(1), "key and value must have the cache's heads");
  OP_CHECK(is_value(key) && key.scalar_type() == value.scalar_type(),
           "key and value must both be float32, bfloat16 or float16");
  OP_CHECK(key.stride(2) == 1 && value.stride(2) == 1,
           "key and value must have stride 1 in their last dimension");
  OP_CHECK(slot_mapping.dim() == 1 && slot_mapping.size(0) == T &&
               slot_mapping.scalar_type() == ScalarType::Long && slot_mapping.is_contiguous(),
           "slot_mapping must be contiguous int64 [T]");
  for (const Tensor* t : {&value, &k_cache, &v_cache, &k_scale, &v_scale, &slot_mapping})
    OP_CHECK(t->device() == key.device(), "all tensors must be on the device of key");
  OP_CHECK(!overlaps_itself(k_cache) && !overlaps_itself(v_cache),
           "k_cache and v_cache must not overlap themselves");
  const Span s_k = span_of(op, k_cache), s_v = span_of(op, v_cache);
  const Span s_ks = span_of(op, k_scale), s_vs = span_of(op, v_scale);
  OP_CHECK(!overlap(s_k, s_v) || !SharedElement::of(k_cache, v_cache),
           "k_cache and v_cache must share no memory");
  OP_CHECK(!overlap(s_ks, s_vs) && !overlap(s_k, s_ks) && !overlap(s_k, s_vs) &&
               !overlap(s_v, s_ks) && !overlap(s_v, s_vs),
           "the scales must not overlap each other or the cache");
  for (const Tensor* t : {&key, &value, &slot_mapping}) {
    const Span s = span_of(op, *t);
    OP_CHECK(!overlap(s_k, s) && !overlap(s_v, s) && !overlap(s_ks, s) && !overlap(s_vs, s),
             "the cache must not overlap an input");
  }
  OP_CHECK(fits32(T) && cache_fits32(k_cache), "a size exceeds int32");
  check_on_gpu(op, key);
  const c10::hip::HIPGuardMasqueradingAsCUDA guard(key.device());
  PthAttnWriteF8Args a{};
  a.abi_version = PTH_ATTN_ABI_VERSION;
  a.struct_bytes = static_cast<int32_t>(sizeof(PthAttnWriteF8Args));
  a.cache = cache_of(k_cache, v_cache, k_scale, v_scale);
  a.key = key.data_ptr();
  a.value = value.data_ptr();
  a.key_stride_token = byte_stride(key, 0);
  a.key_stride_head = byte_stride(key, 1);
  a.value_stride_token = byte_stride(value, 0);
  a.value_stride_head = byte_stride(value, 1);
  a.slot_mapping = static_cast<const int64_t*>(slot_mapping.data_ptr());
  a.kv_dtype = dtype_code(key.scalar_type());
  a.num_tokens = static_cast<int32_t>(T);
  const int32_t rc = pa::launch_write_f8(a, stream_of_device(key));
  OP_CHECK(rc == PTH_ATTN_OK, pa::last_error());
}

void gather_cache_fp8(const Tensor& key, const Tensor& value, const Tensor& k_cache,
                      const Tensor& v_cache, const Tensor& k_scale, const Tensor& v_scale,
                      const Tensor& block_table, const Tensor& row_start_loc,
                      const std::optional<Tensor>& first) {
  const char* op = "gather_cache_fp8";
  OP_CHECK(key.dim() == 3 && value.dim() == 3, "key and value must be 3-D [T, Hkv, D]");
  OP_CHECK(key.sizes() == value.sizes(), "key and value must have the same shape");
  const int64_t T = key.size(0);
  check_cache_f8(op, k_cache, v_cache, k_scale, v_scale, key.size(2));
  OP_CHECK(k_cache.size(2) == key.size(1), "key and value must have the cache's heads");
  OP_CHECK(is_value(key) && key.scalar_type() == value.scalar_type(),
           "key and value must both be float32, bfloat16 or float16");
  OP_CHECK(key.stride(2) == 1 && value.stride(2) == 1,
           "key and value must have stride 1 in their last dimension");
  OP_CHECK(row_start_loc.dim() == 1 && row_start_loc.scalar_type() == ScalarType::Int &&
               row_start_loc.is_contiguous() && row_start_loc.size(0) >= 1,
           "row_start_loc must be contiguous int32 [num_reqs + 1]");
  const int64_t R = row_start_loc.size(0) - 1;
  OP_CHECK(block_table.dim() == 2 && block_table.scalar_type() == ScalarType::Int &&
               block_table.stride(1) == 1 && block_table.size(0) >= R,
           "block_table must be int32 [>= num_reqs, max_blocks] with stride 1 in its last "
           "dimension");
  OP_CHECK(!first.has_value() || (first->dim() == 1 && first->scalar_type() == ScalarType::Int &&
                                  first->is_contiguous() && first->size(0) == R),
           "first must be contiguous int32 [num_reqs]");
  for (const Tensor* t : {&value, &k_cache, &v_cache, &k_scale, &v_scale, &block_table,
                          &row_start_loc})
    OP_CHECK(t->device() == key.device(), "all tensors must be on the device of key");
  OP_CHECK(!first.has_value() || first->device() == key.device(),
           "all tensors must be on the device of key");
  OP_CHECK(!overlaps_itself(key) && !overlaps_itself(value),
           "key and value must not overlap themselves");
  const Span s_k = span_of(op, key), s_v = span_of(op, value);
  OP_CHECK(!overlap(s_k, s_v) || !SharedElement::of(key, value),
           "key and value must share no memory");
  for (const Tensor* t : {&k_cache, &v_cache, &k_scale, &v_scale, &block_table, &row_start_loc}) {
    const Span s = span_of(op, *t);
    OP_CHECK(!overlap(s_k, s) && !overlap(s_v, s), "an output must not overlap an input");
  }
  if (first.has_value()) {
    const Span s = span_of(op, *first);
    OP_CHECK(!overlap(s_k, s) && !overlap(s_v, s), "an output must not overlap an input");
  }
  OP_CHECK(fits32(T) && cache_fits32(k_cache) && fits32(R) && fits32(block_table.size(1)),
           "a size exceeds int32");
  check_on_gpu(op, key);
  const c10::hip::HIPGuardMasqueradingAsCUDA guard(key.device());
  PthAttnGatherF8Args a{};
  a.abi_version = PTH_ATTN_ABI_VERSION;
  a.struct_bytes = static_cast<int32_t>(sizeof(PthAttnGatherF8Args));
  a.cache = cache_of(k_cache, v_cache, k_scale, v_scale);
  a.key = key.data_ptr();
  a.value = value.data_ptr();
  a.key_stride_token = byte_stride(key, 0);
  a.key_stride_head = byte_stride(key, 1);
  a.value_stride_token = byte_stride(value, 0);
  a.value_stride_head = byte_stride(value, 1);
  a.block_table = static_cast<const int32_t*>(block_table.data_ptr());
  a.block_table_row_stride = block_table.stride(0);
  a.row_start_loc = static_cast<const int32_t*>(row_start_loc.data_ptr());
  a.first = first.has_value() ? static_cast<const int32_t*>(first->data_ptr()) : nullptr;
  a.block_table_width = static_cast<int32_t>(block_table.size(1));
  a.num_reqs = static_cast<int32_t>(R);
  a.kv_dtype = dtype_code(key.scalar_type());
  a.num_tokens = static_cast<int32_t>(T);
  const int32_t rc = pa::launch_gather_f8(a, stream_of_device(key));
  OP_CHECK(rc == PTH_ATTN_OK, pa::last_error());
}

// ---- attention ------------------------------------------------------------

void paged_attn_fp8_fwd(const Tensor& out, const Tensor& q, const Tensor& k_cache,
                        const Tensor& v_cache, const Tensor& k_scale, const Tensor& v_scale,
                        const Tensor& block_table, const Tensor& seq_lens,
                        const std::optional<Tensor>& query_start_loc, int64_t max_query_len,
                        int64_t max_seq_len, double softmax_scale, const Tensor& ws,
                        int64_t window, bool causal) {
  const char* op = "paged_attn_fp8_fwd";
  OP_CHECK(q.dim() == 3, "q must be 3-D [T, Hq, D], got ", q.dim(), "-D");
  OP_CHECK(is16(q), "q must be bfloat16 or float16");
  const int64_t T = q.size(0), Hq = q.size(1), D = q.size(2);
  OP_CHECK(q.stride(2) == 1, "q must have stride 1 in its last dimension");
  OP_CHECK(out.dim() == 3 && out.sizes() == q.sizes() && out.scalar_type() == q.scalar_type(),
           "out must have the shape and dtype of q");
  OP_CHECK(out.stride(2) == 1, "out must have stride 1 in its last dimension");
  check_cache_f8(op, k_cache, v_cache, k_scale, v_scale, D);
  const int64_t Hkv = k_cache.size(2);
  OP_CHECK(Hq >= 1 && Hq % Hkv == 0, "Hq = ", Hq, " must be a positive multiple of Hkv = ", Hkv);
  OP_CHECK(Hq / Hkv <= 64, "G = Hq/Hkv = ", Hq / Hkv, " exceeds the supported maximum 64");
  OP_CHECK(seq_lens.dim() == 1 && seq_lens.scalar_type() == ScalarType::Int,
           "seq_lens must be int32 [num_reqs]");
  const int64_t R = seq_lens.size(0);
  OP_CHECK(block_table.dim() == 2 && block_table.scalar_type() == ScalarType::Int,
           "block_table must be int32 [num_reqs, max_blocks]");
  OP_CHECK(block_table.size(0) >= R, "block_table has ", block_table.size(0),
           " rows, fewer than num_reqs = ", R);
  OP_CHECK(seq_lens.stride(0) == 1 && block_table.stride(1) == 1,
           "seq_lens and block_table must have stride 1 in their last dimension");
  if (query_start_loc.has_value()) {
    OP_CHECK(query_start_loc->dim() == 1 && query_start_loc->scalar_type() == ScalarType::Int &&
                 query_start_loc->size(0) == R + 1 && query_start_loc->stride(0) == 1,
             "query_start_loc must be contiguous int32 [num_reqs + 1]");
  } else {
    OP_CHECK(T == R, "q must have one token per request: T = ", T, ", num_reqs = ", R);
  }
  OP_CHECK(max_query_len >= 0, "max_query_len must be >= 0, got ", max_query_len);
  OP_CHECK(max_seq_len >= 0, "max_seq_len must be >= 0, got ", max_seq_len);
  OP_CHECK(std::isfinite(softmax_scale) && softmax_scale > 0.0,
           "softmax_scale must be finite and > 0, got ", softmax_scale);
  OP_CHECK(window >= 0, "window must be >= 0, got ", window);
  OP_CHECK(window == 0 || causal, "a window needs causal");
  OP_CHECK(ws.scalar_type() == ScalarType::Float && ws.dim() == 1 && ws.is_contiguous(),
           "ws must be contiguous float32 [n]");
  for (const Tensor* t : {&out, &k_cache, &v_cache, &k_scale, &v_scale, &block_table, &seq_lens, &ws})
    OP_CHECK(t->device() == q.device(), "all tensors must be on the device of q");
  OP_CHECK(!query_start_loc.has_value() || query_start_loc->device() == q.device(),
           "all tensors must be on the device of q");
  OP_CHECK(!overlaps_itself(out), "out must not overlap itself");
  const Span s_out = span_of(op, out), s_ws = span_of(op, ws), s_q = span_of(op, q);
  OP_CHECK(!overlap(s_out, s_ws), "out and ws must not overlap");
  OP_CHECK(!overlap(s_ws, s_q), "ws must not overlap an input");
  OP_CHECK(!overlap(s_out, s_q) || same_view(out, q) || !SharedElement::of(out, q),
           "out must be q itself or share no memory with it");
  for (const Tensor* t : {&k_cache, &v_cache, &k_scale, &v_scale, &block_table, &seq_lens}) {
    const Span s = span_of(op, *t);
    OP_CHECK(!overlap(s_out, s), "out must not overlap an input");
    OP_CHECK(!overlap(s_ws, s), "ws must not overlap an input");
  }
  if (query_start_loc.has_value()) {
    const Span s = span_of(op, *query_start_loc);
    OP_CHECK(!overlap(s_out, s), "out must not overlap an input");
    OP_CHECK(!overlap(s_ws, s), "ws must not overlap an input");
  }
  OP_CHECK(fits32(T) && fits32(Hq) && cache_fits32(k_cache) && fits32(block_table.size(1)),
           "a size exceeds int32");
  check_on_gpu(op, q);
  const c10::hip::HIPGuardMasqueradingAsCUDA guard(q.device());
  PthAttnPagedF8Args a{};
  a.abi_version = PTH_ATTN_ABI_VERSION;
  a.struct_bytes = static_cast<int32_t>(sizeof(PthAttnPagedF8Args));
  a.cache = cache_of(k_cache, v_cache, k_scale, v_scale);
  a.q = q.data_ptr();
  a.q_stride_token = byte_stride(q, 0);
  a.q_stride_head = byte_stride(q, 1);
  a.out = out.data_ptr();
  a.out_stride_token = byte_stride(out, 0);
  a.out_stride_head = byte_stride(out, 1);
  a.block_table = static_cast<const int32_t*>(block_table.data_ptr());
  a.block_table_row_stride = block_table.stride(0);
  a.kv_lens = static_cast<const int32_t*>(seq_lens.data_ptr());
  a.query_start_loc = query_start_loc.has_value()
                          ? static_cast<const int32_t*>(query_start_loc->data_ptr())
                          : nullptr;
  a.block_table_width = static_cast<int32_t>(block_table.size(1));
  a.max_kv_len = static_cast<int32_t>(std::min<int64_t>(max_seq_len, INT32_MAX));
  a.dtype = dtype_code(q.scalar_type());
  a.num_reqs = static_cast<int32_t>(R);
  a.num_tokens = static_cast<int32_t>(T);
  a.num_q_heads = static_cast<int32_t>(Hq);
  a.max_query_len = static_cast<int32_t>(std::min<int64_t>(max_query_len, INT32_MAX));
  a.window = static_cast<int32_t>(std::min<int64_t>(window, INT32_MAX));
  a.causal = causal ? 1 : 0;
  a.softmax_scale = static_cast<float>(softmax_scale);
  a.ws = static_cast<float*>(ws.data_ptr());
  a.ws_floats = ws.numel();
  const int32_t rc = pa::launch_paged_f8(a, stream_of_device(q));
  OP_CHECK(rc == PTH_ATTN_OK, pa::last_error());
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(pth_flash_attn, m) {
  m.def(
      "rotary_embedding(Tensor! q_out, Tensor! k_out, Tensor q, Tensor k, Tensor positions, "
      "Tensor turns, bool interleaved=False, float scale=1.0, bool inverse=False) -> ()");
  m.def(
      "reshape_and_cache_fp8(Tensor key, Tensor value, Tensor! k_cache, Tensor! v_cache, "
      "Tensor! k_scale, Tensor! v_scale, Tensor slot_mapping) -> ()");
  m.def(
      "gather_cache_fp8(Tensor! key, Tensor! value, Tensor k_cache, Tensor v_cache, "
      "Tensor k_scale, Tensor v_scale, Tensor block_table, Tensor row_start_loc, "
      "Tensor? first=None) -> ()");
  m.def(
      "paged_attn_fp8_fwd(Tensor! out, Tensor q, Tensor k_cache, Tensor v_cache, "
      "Tensor k_scale, Tensor v_scale, Tensor block_table, Tensor seq_lens, "
      "Tensor? query_start_loc, int max_query_len, int max_seq_len, float softmax_scale, "
      "Tensor! ws, int window=0, bool causal=True) -> ()");
}

TORCH_LIBRARY_IMPL(pth_flash_attn, CUDA, m) {
  m.impl("rotary_embedding", &rotary_embedding);
  m.impl("reshape_and_cache_fp8", &reshape_and_cache_fp8);
  m.impl("gather_cache_fp8", &gather_cache_fp8);
  m.impl("paged_attn_fp8_fwd", &paged_attn_fp8_fwd);
}

// Validates, then raises: CPU tensors exist only to test the checks.
TORCH_LIBRARY_IMPL(pth_flash_attn, CPU, m) {
  m.impl("rotary_embedding", &rotary_embedding);
  m.impl("reshape_and_cache_fp8", &reshape_and_cache_fp8);
  m.impl("gather_cache_fp8", &gather_cache_fp8);
  m.impl("paged_attn_fp8_fwd", &paged_attn_fp8_fwd);
}
