// torch_op_p16.cpp -- the torch ops around a paged cache in the model's own
// 16-bit type: build_step_tables, reshape_and_cache_16bit, paged_decode_fwd
// and cross_attn_fwd (no counterparts in the reference). As in torch_op.cpp,
// the CUDA key (HIP tensors on ROCm torch) checks and launches, on the current
// stream of the tensors' device, allocating nothing and reading nothing back;
// the CPU key checks and raises. The fakes in ops.py make the same metadata
// checks with the same messages.

#include "p16.h"
#include "torch_checks.h"

namespace {

// ---- attention ------------------------------------------------------------

// A cache view pair for heads of D values of type `dtype`.
void check_cache(const char* op, const Tensor& k, const Tensor& v, int64_t D, ScalarType dtype) {
  OP_CHECK(k.dim() == 4 && v.dim() == 4 && k.sizes() == v.sizes() && k.size(3) == D,
           "k_cache and v_cache must be [num_blocks, block_size, Hkv, ", D, "]");
  OP_CHECK(k.scalar_type() == dtype && v.scalar_type() == dtype,
           "k_cache and v_cache must have the dtype of q");
  OP_CHECK(k.size(0) >= 1 && k.size(1) >= 1 && k.size(2) >= 1,
           "k_cache and v_cache must not be empty");
  OP_CHECK(k.stride(3) == 1 && v.stride(3) == 1,
           "k_cache and v_cache must have stride 1 in their last dimension");
}

// Checks without data pointers, shared by the two attention ops (the fake in
// ops.py runs the same list with the same messages).
void check_attention(const char* op, const char* lens_name, const Tensor& out, const Tensor& q,
                     const Tensor& k_cache, const Tensor& v_cache, const Tensor& block_table,
                     const Tensor& lens, const Tensor* query_start_loc, int64_t max_len,
                     double softmax_scale, const Tensor& ws, int64_t window) {
  OP_CHECK(q.dim() == 3, "q must be 3-D [T, Hq, D], got ", q.dim(), "-D");
  OP_CHECK(is16(q), "q must be bfloat16 or float16");
  const int64_t T = q.size(0), Hq = q.size(1), D = q.size(2);
  OP_CHECK(D == 64 || D == 128 || D == 256, "head size D = q.size(2) must be 64, 128 or 256, got ",
           D);
  OP_CHECK(q.stride(2) == 1, "q must have stride 1 in its last dimension");
  OP_CHECK(out.dim() == 3 && out.sizes() == q.sizes() && out.scalar_type() == q.scalar_type(),
           "out must have the shape and dtype of q");
  OP_CHECK(out.stride(2) == 1, "out must have stride 1 in its last dimension");
  check_cache(op, k_cache, v_cache, D, q.scalar_type());
  const int64_t Hkv = k_cache.size(2);
  OP_CHECK(Hq >= 1 && Hq % Hkv == 0, "Hq = ", Hq, " must be a positive multiple of Hkv = ", Hkv);
  OP_CHECK(Hq / Hkv <= 64, "G = Hq/Hkv = ", Hq / Hkv, " exceeds the supported maximum 64");
  OP_CHECK(lens.dim() == 1 && lens.scalar_type() == ScalarType::Int, lens_name,
           " must be int32 [num_reqs]");
  const int64_t R = lens.size(0);
  OP_CHECK(block_table.dim() == 2 && block_table.scalar_type() == ScalarType::Int,
           "block_table must be int32 [num_reqs, max_blocks]");
  OP_CHECK(block_table.size(0) >= R, "block_table has ", block_table.size(0),
           " rows, fewer than num_reqs = ", R);
  OP_CHECK(lens.stride(0) == 1 && block_table.stride(1) == 1, lens_name,
           " and block_table must have stride 1 in their last dimension");
  if (query_start_loc != nullptr) {
    OP_CHECK(query_start_loc->dim() == 1 && query_start_loc->scalar_type() == ScalarType::Int &&
                 query_start_loc->size(0) == R + 1 && query_start_loc->stride(0) == 1,
             "query_start_loc must be contiguous int32 [num_reqs + 1]");
  } else {
    OP_CHECK(T == R, "q must have one token per request: T = ", T, ", num_reqs = ", R);
  }
  OP_CHECK(max_len >= 0, lens_name, "' bound must be >= 0, got ", max_len);
  OP_CHECK(std::isfinite(softmax_scale) && softmax_scale > 0.0,
           "softmax_scale must be finite and > 0, got ", softmax_scale);
  OP_CHECK(window >= 0, "window must be >= 0, got ", window);
  OP_CHECK(ws.scalar_type() == ScalarType::Float && ws.dim() == 1 && ws.is_contiguous(),
           "ws must be contiguous float32 [n]");
  for (const Tensor* t : {&out, &k_cache, &v_cache, &block_table, &lens, &ws})
    OP_CHECK(t->device() == q.device(), "all tensors must be on the device of q");
  OP_CHECK(query_start_loc == nullptr || query_start_loc->device() == q.device(),
           "all tensors must be on the device of q");
}

void attend(const char* op, const char* lens_name, const Tensor& out, const Tensor& q,
            const Tensor& k_cache, const Tensor& v_cache, const Tensor& block_table,
            const Tensor& lens, const Tensor* query_start_loc, int64_t max_query_len,
            int64_t max_len, double softmax_scale, const Tensor& ws, int64_t window) {
  check_attention(op, lens_name, out, q, k_cache, v_cache, block_table, lens, query_start_loc,
                  max_len, softmax_scale, ws, window);
  OP_CHECK(!overlaps_itself(out), "out must not overlap itself");
  const Span s_out = span_of(op, out), s_ws = span_of(op, ws), s_q = span_of(op, q);
  OP_CHECK(!overlap(s_out, s_ws), "out and ws must not overlap");
  OP_CHECK(!overlap(s_ws, s_q), "ws must not overlap an input");
  OP_CHECK(!overlap(s_out, s_q) || same_view(out, q) || !SharedElement::of(out, q),
           "out must be q itself or share no memory with it");
  for (const Tensor* t : {&k_cache, &v_cache, &block_table, &lens}) {
    const Span s = span_of(op, *t);
    OP_CHECK(!overlap(s_out, s), "out must not overlap an input");
    OP_CHECK(!overlap(s_ws, s), "ws must not overlap an input");
  }
  if (query_start_loc != nullptr) {
    const Span s = span_of(op, *query_start_loc);
    OP_CHECK(!overlap(s_out, s), "out must not overlap an input");
    OP_CHECK(!overlap(s_ws, s), "ws must not overlap an input");
  }
  OP_CHECK(fits32(q.size(0)) && fits32(q.size(1)) && fits32(k_cache.size(0)) &&
               fits32(k_cache.size(1)) && fits32(block_table.size(1)),
           "a size exceeds int32");
  check_on_gpu(op, q);
  const c10::hip::HIPGuardMasqueradingAsCUDA guard(q.device());
  PthAttnP16Args a{};
  a.abi_version = PTH_ATTN_ABI_VERSION;
  a.struct_bytes = static_cast<int32_t>(sizeof(PthAttnP16Args));
  a.q = q.data_ptr();
  a.q_stride_token = byte_stride(q, 0);
  a.q_stride_head = byte_stride(q, 1);
  a.out = out.data_ptr();
  a.out_stride_token = byte_stride(out, 0);
  a.out_stride_head = byte_stride(out, 1);
  a.dtype = dtype_code(q.scalar_type());
  a.num_blocks = static_cast<int32_t>(k_cache.size(0));
  a.block_size = static_cast<int32_t>(k_cache.size(1));
  a.num_kv_heads = static_cast<int32_t>(k_cache.size(2));
  a.head_size = static_cast<int32_t>(q.size(2));
  a.k_cache = stream_of(k_cache);
  a.v_cache = stream_of(v_cache);
  a.block_table = static_cast<const int32_t*>(block_table.data_ptr());
  a.block_table_row_stride = block_table.stride(0);
  a.block_table_width = static_cast<int32_t>(block_table.size(1));
  a.max_kv_len = static_cast<int32_t>(std::min<int64_t>(max_len, INT32_MAX));
  a.kv_lens = static_cast<const int32_t*>(lens.data_ptr());
  a.query_start_loc =
      query_start_loc ? static_cast<const int32_t*>(query_start_loc->data_ptr()) : nullptr;
  a.num_reqs = static_cast<int32_t>(lens.size(0));
  a.num_tokens = static_cast<int32_t>(q.size(0));
  a.num_q_heads = static_cast<int32_t>(q.size(1));
  a.max_query_len = static_cast<int32_t>(std::min<int64_t>(max_query_len, INT32_MAX));
  a.window = static_cast<int32_t>(std::min<int64_t>(window, INT32_MAX - 1024));
  a.softmax_scale = static_cast<float>(softmax_scale);
  a.ws = static_cast<float*>(ws.data_ptr());
  a.ws_floats = ws.numel();
  const int32_t rc = pa::launch_p16(a, stream_of_device(q));
  OP_CHECK(rc == PTH_ATTN_OK, pa::last_error());
}

void paged_decode_fwd(const Tensor& out, const Tensor& q, const Tensor& k_cache,
                      const Tensor& v_cache, const Tensor& block_table, const Tensor& seq_lens,
                      int64_t max_seq_len, double softmax_scale, const Tensor& ws,
                      int64_t window) {
  attend("paged_decode_fwd", "seq_lens", out, q, k_cache, v_cache, block_table, seq_lens, nullptr,
         1, max_seq_len, softmax_scale, ws, window);
}

void cross_attn_fwd(const Tensor& out, const Tensor& q, const Tensor& k_cache,
                    const Tensor& v_cache, const Tensor& block_table, const Tensor& encoder_lens,
                    const Tensor& query_start_loc, int64_t max_query_len, int64_t max_encoder_len,
                    double softmax_scale, const Tensor& ws) {
  const char* op = "cross_attn_fwd";
  OP_CHECK(max_query_len >= 0, "max_query_len must be >= 0, got ", max_query_len);
  attend(op, "encoder_lens", out, q, k_cache, v_cache, block_table, encoder_lens,
         &query_start_loc, max_query_len, max_encoder_len, softmax_scale, ws, 0);
}

// ---- cache writer ---------------------------------------------------------

void reshape_and_cache_16bit(const Tensor& key, const Tensor& value, const Tensor& k_cache,
                             const Tensor& v_cache, const Tensor& slot_mapping) {
  const char* op = "reshape_and_cache_16bit";
  OP_CHECK(key.dim() == 3 && value.dim() == 3, "key and value must be 3-D [T, Hkv, D]");
  OP_CHECK(key.sizes() == value.sizes(), "key and value must have the same shape");
  const int64_t T = key.size(0), Hkv = key.size(1), D = key.size(2);
  OP_CHECK(D == 64 || D == 128 || D == 256, "head size must be 64, 128 or 256, got ", D);
  OP_CHECK(k_cache.dim() == 4 && v_cache.dim() == 4 && k_cache.sizes() == v_cache.sizes() &&
               k_cache.size(2) == Hkv && k_cache.size(3) == D,
           "k_cache and v_cache must be [num_blocks, block_size, ", Hkv, ", ", D, "]");
  OP_CHECK(is16(k_cache) && k_cache.scalar_type() == v_cache.scalar_type(),
           "k_cache and v_cache must both be bfloat16 or float16");
  OP_CHECK(k_cache.size(0) >= 1 && k_cache.size(1) >= 1 && Hkv >= 1,
           "k_cache and v_cache must not be empty");
  OP_CHECK(key.scalar_type() == value.scalar_type() &&
               (key.scalar_type() == ScalarType::Float ||
                key.scalar_type() == k_cache.scalar_type()),
           "key and value must both be float32 or have the dtype of the cache");
  OP_CHECK(key.stride(2) == 1 && value.stride(2) == 1 && k_cache.stride(3) == 1 &&
               v_cache.stride(3) == 1,
           "key, value, k_cache and v_cache must have stride 1 in their last dimension");
  OP_CHECK(slot_mapping.dim() == 1 && slot_mapping.size(0) == T &&
               slot_mapping.scalar_type() == ScalarType::Long && slot_mapping.is_contiguous(),
           "slot_mapping must be contiguous int64 [T]");
  for (const Tensor* t : {&value, &k_cache, &v_cache, &slot_mapping})
    OP_CHECK(t->device() == key.device(), "all tensors must be on the device of key");
  OP_CHECK(!overlaps_itself(k_cache) && !overlaps_itself(v_cache),
           "k_cache and v_cache must not overlap themselves");
  const Span s_k = span_of(op, k_cache), s_v = span_of(op, v_cache);
  OP_CHECK(!overlap(s_k, s_v) || !SharedElement::of(k_cache, v_cache) ||
               (same_view(k_cache, v_cache) && same_view(key, value)),
           "k_cache and v_cache must share no memory, unless both are one view and so are key "
           "and value");
  for (const Tensor* t : {&key, &value, &slot_mapping}) {
    const Span s = span_of(op, *t);
    OP_CHECK(!overlap(s_k, s) && !overlap(s_v, s), "the cache must not overlap an input");
  }
  OP_CHECK(fits32(T) && fits32(k_cache.size(0)) && fits32(k_cache.size(1)) && fits32(Hkv),
           "a size exceeds int32");
  check_on_gpu(op, key);
  const c10::hip::HIPGuardMasqueradingAsCUDA guard(key.device());
  PthAttnWrite16Args a{};
  a.abi_version = PTH_ATTN_ABI_VERSION;
  a.struct_bytes = static_cast<int32_t>(sizeof(PthAttnWrite16Args));
  a.key = key.data_ptr();
  a.value = value.data_ptr();
  a.key_stride_token = byte_stride(key, 0);
  a.key_stride_head = byte_stride(key, 1);
  a.value_stride_token = byte_stride(value, 0);
  a.value_stride_head = byte_stride(value, 1);
  a.kv_dtype = dtype_code(key.scalar_type());
  a.cache_dtype = dtype_code(k_cache.scalar_type());
  a.num_tokens = static_cast<int32_t>(T);
  a.num_kv_heads = static_cast<int32_t>(Hkv);
  a.head_size = static_cast<int32_t>(D);
  a.block_size = static_cast<int32_t>(k_cache.size(1));
  a.num_blocks = static_cast<int32_t>(k_cache.size(0));
  a.slot_mapping = static_cast<const int64_t*>(slot_mapping.data_ptr());
  a.k_cache = stream_of(k_cache);
  a.v_cache = stream_of(v_cache);
  const int32_t rc = pa::launch_write_kv16(a, stream_of_device(key));
  OP_CHECK(rc == PTH_ATTN_OK, pa::last_error());
}

// ---- step tables ----------------------------------------------------------

void build_step_tables(const Tensor& block_table, const Tensor& slot_mapping,
                       const Tensor& seq_lens, const Tensor& query_start_loc,
                       const Tensor& pool_out, const Tensor& context_lens,
                       const Tensor& query_lens, const Tensor& free_pages, const Tensor& pool_in,
                       int64_t block_size) {
  const char* op = "build_step_tables";
  const auto ints = [&](const Tensor& t, int64_t n, const char* name) {
    OP_CHECK(t.dim() == 1 && t.scalar_type() == ScalarType::Int && t.is_contiguous() &&
                 (n < 0 || t.size(0) == n),
             name, " must be contiguous int32 [", n < 0 ? "n" : std::to_string(n), "]");
  };
  ints(context_lens, -1, "context_lens");
  const int64_t R = context_lens.size(0);
  ints(query_lens, R, "query_lens");
  ints(seq_lens, R, "seq_lens");
  ints(query_start_loc, R + 1, "query_start_loc");
  ints(free_pages, -1, "free_pages");
  ints(pool_in, 2, "pool_in");
  ints(pool_out, 2, "pool_out");
  OP_CHECK(block_table.dim() == 2 && block_table.scalar_type() == ScalarType::Int &&
               block_table.stride(1) == 1 && block_table.size(0) >= R,
           "block_table must be int32 [>= num_reqs, max_blocks] with stride 1 in its last "
           "dimension");
  OP_CHECK(!overlaps_itself(block_table), "the rows of block_table must not overlap");
  OP_CHECK(slot_mapping.dim() == 1 && slot_mapping.scalar_type() == ScalarType::Long &&
               slot_mapping.is_contiguous(),
           "slot_mapping must be contiguous int64 [T]");
  OP_CHECK(block_size >= 1, "block_size must be >= 1, got ", block_size);
  OP_CHECK(fits32(R) && fits32(block_table.size(1)) && fits32(block_size), "a size exceeds int32");
  const Tensor* outs[] = {&block_table, &slot_mapping, &seq_lens, &query_start_loc, &pool_out};
  const Tensor* ins[] = {&context_lens, &query_lens, &free_pages, &pool_in};
  for (const Tensor* t : outs)
    OP_CHECK(t->device() == context_lens.device(),
             "all tensors must be on the device of context_lens");
  for (const Tensor* t : ins)
    OP_CHECK(t->device() == context_lens.device(),
             "all tensors must be on the device of context_lens");
  Span s[9];
  for (size_t i = 0; i < 5; ++i) s[i] = span_of(op, *outs[i]);
  for (size_t i = 0; i < 4; ++i) s[5 + i] = span_of(op, *ins[i]);
  for (size_t i = 0; i < 5; ++i) {
    for (size_t j = i + 1; j < 5; ++j)
      OP_CHECK(!overlap(s[i], s[j]), "the outputs must not overlap each other");
    for (size_t j = 5; j < 9; ++j)
      OP_CHECK(!overlap(s[i], s[j]), "an output must not overlap an input");
  }
  check_on_gpu(op, context_lens);
  const c10::hip::HIPGuardMasqueradingAsCUDA guard(context_lens.device());
  PthAttnTablesArgs a{};
  a.abi_version = PTH_ATTN_ABI_VERSION;
  a.struct_bytes = static_cast<int32_t>(sizeof(PthAttnTablesArgs));
  a.block_table = static_cast<int32_t*>(block_table.data_ptr());
  a.block_table_row_stride = block_table.stride(0);
  a.block_table_width = static_cast<int32_t>(block_table.size(1));
  a.block_size = static_cast<int32_t>(block_size);
  a.slot_mapping = static_cast<int64_t*>(slot_mapping.data_ptr());
  a.num_slots = slot_mapping.size(0);
  a.seq_lens = static_cast<int32_t*>(seq_lens.data_ptr());
  a.query_start_loc = static_cast<int32_t*>(query_start_loc.data_ptr());
  a.pool_out = static_cast<int32_t*>(pool_out.data_ptr());
  a.context_lens = static_cast<const int32_t*>(context_lens.data_ptr());
  a.query_lens = static_cast<const int32_t*>(query_lens.data_ptr());
  a.free_pages = static_cast<const int32_t*>(free_pages.data_ptr());
  a.num_free = free_pages.size(0);
  a.pool_in = static_cast<const int32_t*>(pool_in.data_ptr());
  a.num_reqs = static_cast<int32_t>(R);
  const int32_t rc = pa::launch_step_tables(a, stream_of_device(context_lens));
  OP_CHECK(rc == PTH_ATTN_OK, pa::last_error());
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(pth_flash_attn, m) {
  m.def(
      "build_step_tables(Tensor! block_table, Tensor! slot_mapping, Tensor! seq_lens, "
      "Tensor! query_start_loc, Tensor! pool_out, Tensor context_lens, Tensor query_lens, "
      "Tensor free_pages, Tensor pool_in, int block_size) -> ()");
  m.def(
      "reshape_and_cache_16bit(Tensor key, Tensor value, Tensor! k_cache, Tensor! v_cache, "
      "Tensor slot_mapping) -> ()");
  m.def(
      "paged_decode_fwd(Tensor! out, Tensor q, Tensor k_cache, Tensor v_cache, "
      "Tensor block_table, Tensor seq_lens, int max_seq_len, float softmax_scale, Tensor! ws, "
      "int window=0) -> ()");
  m.def(
      "cross_attn_fwd(Tensor! out, Tensor q, Tensor k_cache, Tensor v_cache, "
      "Tensor block_table, Tensor encoder_lens, Tensor query_start_loc, int max_query_len, "
      "int max_encoder_len, float softmax_scale, Tensor! ws) -> ()");
}

TORCH_LIBRARY_IMPL(pth_flash_attn, CUDA, m) {
  m.impl("build_step_tables", &build_step_tables);
  m.impl("reshape_and_cache_16bit", &reshape_and_cache_16bit);
  m.impl("paged_decode_fwd", &paged_decode_fwd);
  m.impl("cross_attn_fwd", &cross_attn_fwd);
}

// Validates, then raises: CPU tensors exist only to test the checks.
TORCH_LIBRARY_IMPL(pth_flash_attn, CPU, m) {
  m.impl("build_step_tables", &build_step_tables);
  m.impl("reshape_and_cache_16bit", &reshape_and_cache_16bit);
  m.impl("paged_decode_fwd", &paged_decode_fwd);
  m.impl("cross_attn_fwd", &cross_attn_fwd);
}
