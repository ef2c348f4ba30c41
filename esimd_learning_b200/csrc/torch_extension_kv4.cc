// torch_extension_kv4.cc — torch.library registration of the paged 4-bit
// key/value cache ops (plan, append, gather, attention) on the CUDA dispatch
// key.  No reference counterpart.  As in torch_extension.cc each op checks its
// tensors and forwards raw pointers and the current stream to the C ABI.
#include <Python.h>

#include "torch_common.h"

using namespace cek_torch;

namespace {

void check_same_device(const at::Tensor& t, const at::Tensor& like, const char* op, const char* name) {
  TORCH_CHECK(t.is_cuda() && t.device() == like.device(), op, ": ", name, " must be on the device of the first argument");
}

void check_i32(const at::Tensor& t, const at::Tensor& like, const char* op, const char* name) {
  check_same_device(t, like, op, name);
  TORCH_CHECK(t.scalar_type() == at::kInt && t.is_contiguous(), op, ": ", name, " must be contiguous int32");
}

void check_i64(const at::Tensor& t, const at::Tensor& like, const char* op, const char* name) {
  check_same_device(t, like, op, name);
  TORCH_CHECK(t.scalar_type() == at::kLong && t.dim() == 1 && t.is_contiguous(), op, ": ", name,
              " must be contiguous int64 [tokens]");
}

// block_table: int32 [requests, width], rows contiguous
void check_table(const at::Tensor& t, const at::Tensor& like, int64_t requests, const char* op) {
  check_same_device(t, like, op, "block_table");
  TORCH_CHECK(t.scalar_type() == at::kInt && t.dim() == 2 && t.size(0) == requests, op,
              ": block_table must be int32 [requests, width]");
  TORCH_CHECK((t.size(1) <= 1 || t.stride(1) == 1) && (requests <= 1 || t.stride(0) >= t.size(1)), op,
              ": block_table rows must be contiguous and not overlap");
}

// The stride of a dimension that has one entry does not matter; a multiple of
// 8 in its place keeps the vector accesses.
int64_t stride_of(const at::Tensor& t, int64_t d, int64_t dense) { return t.size(d) > 1 ? t.stride(d) : dense; }

// [tokens, heads, head_dim], channels contiguous, other strides free
void check_heads(const at::Tensor& t, const at::Tensor& like, int64_t heads, int64_t d, const char* op,
                 const char* name) {
  check_same_device(t, like, op, name);
  TORCH_CHECK(is_half_or_bf16(t), op, ": ", name, " must be fp16 or bf16");
  TORCH_CHECK(t.dim() == 3 && t.size(1) == heads && t.size(2) == d, op, ": ", name,
              " must be [tokens, heads, head_dim]");
  TORCH_CHECK(t.stride(2) == 1, op, ": the channels of ", name, " must be contiguous");
}

cek_kv4_cache make_cache(const at::Tensor& kv_cache, const at::Tensor& kv_scales, int64_t page_size, int64_t head_dim,
                         const char* op) {
  TORCH_CHECK(kv_cache.is_cuda() && kv_cache.scalar_type() == at::kByte && kv_cache.dim() == 3, op,
              ": kv_cache must be a uint8 CUDA tensor [pages, kv_heads, page bytes]");
  const int64_t block = cek_kv4_page_bytes(page_size, head_dim);
  TORCH_CHECK(block > 0, op, ": page_size must be 16, 32, 64 or 128 and head_dim 64, 128 or 256");
  TORCH_CHECK(kv_cache.size(2) == block && kv_cache.stride(2) == 1, op, ": the last dim of kv_cache must be ", block,
              " contiguous bytes");
  check_same_device(kv_scales, kv_cache, op, "kv_scales");
  TORCH_CHECK(kv_scales.scalar_type() == at::kFloat && kv_scales.is_contiguous() && kv_scales.dim() == 2 &&
                  kv_scales.size(0) == 2 && kv_scales.size(1) == kv_cache.size(1),
              op, ": kv_scales must be contiguous fp32 [2, kv_heads]");
  TORCH_CHECK(kv_cache.size(0) > 0 && kv_cache.size(1) > 0, op, ": kv_cache must have at least one page and one kv head");
  cek_kv4_cache c;
  c.data = kv_cache.data_ptr();
  c.scales = kv_scales.data_ptr<float>();
  c.num_pages = kv_cache.size(0);
  c.kv_heads = kv_cache.size(1);
  c.head_stride = stride_of(kv_cache, 1, block);
  c.page_stride = stride_of(kv_cache, 0, block * c.kv_heads);
  c.head_dim = head_dim;
  c.page_size = page_size;
  return c;
}

// key/value of append and gather
void check_pair(const at::Tensor& key, const at::Tensor& value, const at::Tensor& kv_cache, const at::Tensor& slots,
                const char* op) {
  TORCH_CHECK(key.is_cuda() && key.dim() == 3, op, ": key must be a CUDA tensor [tokens, kv_heads, head_dim]");
  TORCH_CHECK(kv_cache.dim() == 3, op, ": kv_cache must be [pages, kv_heads, page bytes]");
  check_heads(key, kv_cache, kv_cache.size(1), key.size(2), op, "key");
  check_heads(value, kv_cache, kv_cache.size(1), key.size(2), op, "value");
  TORCH_CHECK(key.scalar_type() == value.scalar_type() && key.size(0) == value.size(0), op,
              ": key and value must share a dtype and a token count");
  check_i64(slots, kv_cache, op, "slots");
  TORCH_CHECK(slots.numel() == key.size(0), op, ": one slot per token");
}

}  // namespace

// New: pages, slots and positions of one step from request lengths.
at::Tensor esimd_kv_plan(at::Tensor query_lens, at::Tensor context_lens, at::Tensor block_table, at::Tensor free_pages,
                         at::Tensor free_count, int64_t page_size, at::Tensor query_start, at::Tensor seq_lens,
                         at::Tensor free_count_out, at::Tensor positions, at::Tensor slot_mapping) {
  const char* op = "esimd_kv_plan";
  TORCH_CHECK(query_lens.is_cuda(), op, ": query_lens must be a CUDA tensor");
  const int64_t B = query_lens.numel();
  check_i32(query_lens, query_lens, op, "query_lens");
  check_i32(context_lens, query_lens, op, "context_lens");
  check_i32(free_pages, query_lens, op, "free_pages");
  check_i32(free_count, query_lens, op, "free_count");
  check_i32(query_start, query_lens, op, "query_start");
  check_i32(seq_lens, query_lens, op, "seq_lens");
  check_i32(free_count_out, query_lens, op, "free_count_out");
  check_i64(positions, query_lens, op, "positions");
  check_i64(slot_mapping, query_lens, op, "slot_mapping");
  check_table(block_table, query_lens, B, op);
  TORCH_CHECK(B <= CEK_KV_PLAN_MAX_REQUESTS, op, ": at most ", CEK_KV_PLAN_MAX_REQUESTS, " requests");
  TORCH_CHECK(context_lens.numel() == B && seq_lens.numel() == B && query_start.numel() == B + 1, op,
              ": context_lens and seq_lens [requests], query_start [requests + 1]");
  TORCH_CHECK(free_count.numel() == 1 && free_count_out.numel() == 1, op, ": free_count and free_count_out hold one value");
  TORCH_CHECK(positions.numel() == slot_mapping.numel(), op, ": positions and slot_mapping must have one length");
  TORCH_CHECK(page_size >= 1, op, ": page_size must be positive");
  c10::cuda::CUDAGuard guard(query_lens.device());
  check_status(cek_kv_plan(query_lens.data_ptr<int32_t>(), context_lens.data_ptr<int32_t>(),
                           block_table.data_ptr<int32_t>(), free_pages.data_ptr<int32_t>(),
                           free_count.data_ptr<int32_t>(), query_start.data_ptr<int32_t>(),
                           seq_lens.data_ptr<int32_t>(), free_count_out.data_ptr<int32_t>(),
                           positions.data_ptr<int64_t>(), slot_mapping.data_ptr<int64_t>(), B, block_table.size(1),
                           stride_of(block_table, 0, block_table.size(1)), free_pages.numel(), positions.numel(), page_size,
                           stream_of(query_lens)),
               op);
  return slot_mapping;
}

// New: quantise keys and values into the cache's slots.
at::Tensor esimd_kv4_append(at::Tensor key, at::Tensor value, at::Tensor kv_scales, at::Tensor slot_mapping,
                            at::Tensor kv_cache, int64_t page_size) {
  const char* op = "esimd_kv4_append";
  check_pair(key, value, kv_cache, slot_mapping, op);
  const cek_kv4_cache c = make_cache(kv_cache, kv_scales, page_size, key.size(2), op);
  const int64_t d = c.head_dim, row = d * c.kv_heads;
  c10::cuda::CUDAGuard guard(kv_cache.device());
  check_status(cek_kv4_append(key.data_ptr(), value.data_ptr(), slot_mapping.data_ptr<int64_t>(), &c, key.size(0),
                              stride_of(key, 0, row), stride_of(key, 1, d), stride_of(value, 0, row),
                              stride_of(value, 1, d), io_dtype(key), stream_of(kv_cache)),
               op);
  return kv_cache;
}

// New: the 16-bit values that slots of the cache stand for.
void esimd_kv4_gather(at::Tensor kv_cache, at::Tensor kv_scales, at::Tensor slots, at::Tensor key, at::Tensor value,
                      int64_t page_size) {
  const char* op = "esimd_kv4_gather";
  check_pair(key, value, kv_cache, slots, op);
  const cek_kv4_cache c = make_cache(kv_cache, kv_scales, page_size, key.size(2), op);
  const int64_t d = c.head_dim, row = d * c.kv_heads;
  c10::cuda::CUDAGuard guard(kv_cache.device());
  check_status(cek_kv4_gather(&c, slots.data_ptr<int64_t>(), key.data_ptr(), value.data_ptr(), key.size(0),
                              stride_of(key, 0, row), stride_of(key, 1, d), stride_of(value, 0, row),
                              stride_of(value, 1, d), io_dtype(key), stream_of(kv_cache)),
               op);
}

// New: attention of the step's query tokens over the cache.
at::Tensor esimd_kv4_attention(at::Tensor query, at::Tensor kv_cache, at::Tensor kv_scales, at::Tensor block_table,
                               at::Tensor query_start, at::Tensor seq_lens, at::Tensor output, int64_t page_size,
                               double softmax_scale, int64_t max_query_len, int64_t max_seq_len, int64_t window) {
  const char* op = "esimd_kv4_attention";
  TORCH_CHECK(query.is_cuda() && query.dim() == 3, op, ": query must be a CUDA tensor [tokens, q_heads, head_dim]");
  const int64_t hq = query.size(1), d = query.size(2), T = query.size(0);
  const cek_kv4_cache c = make_cache(kv_cache, kv_scales, page_size, d, op);
  check_heads(query, kv_cache, hq, d, op, "query");
  check_heads(output, kv_cache, hq, d, op, "output");
  TORCH_CHECK(output.scalar_type() == query.scalar_type() && output.size(0) == T, op,
              ": output must match query's dtype and shape");
  TORCH_CHECK(hq > 0 && hq % c.kv_heads == 0, op, ": q_heads must be a multiple of kv_heads");
  check_i32(query_start, kv_cache, op, "query_start");
  check_i32(seq_lens, kv_cache, op, "seq_lens");
  const int64_t B = seq_lens.numel();
  TORCH_CHECK(query_start.numel() == B + 1, op, ": query_start must be [requests + 1]");
  check_table(block_table, kv_cache, B, op);
  TORCH_CHECK(max_query_len >= 0 && max_seq_len >= 0 && window >= 0, op,
              ": max_query_len, max_seq_len and window must not be negative");
  TORCH_CHECK(softmax_scale > 0.0, op, ": softmax_scale must be positive");
  c10::cuda::CUDAGuard guard(kv_cache.device());
  const int64_t ws_bytes =
      cek_kv4_attention_workspace_bytes(B, T, hq, c.kv_heads, d, max_query_len, max_seq_len);
  at::Tensor ws;
  if (ws_bytes > 0) ws = at::empty({ws_bytes}, kv_cache.options().dtype(at::kByte));
  check_status(cek_kv4_attention(query.data_ptr(), &c, block_table.data_ptr<int32_t>(), query_start.data_ptr<int32_t>(),
                                 seq_lens.data_ptr<int32_t>(), output.data_ptr(), ws_bytes > 0 ? ws.data_ptr() : nullptr,
                                 ws_bytes, B, T, hq, block_table.size(1), stride_of(block_table, 0, block_table.size(1)),
                                 stride_of(query, 0, hq * d), stride_of(query, 1, d), stride_of(output, 0, hq * d),
                                 stride_of(output, 1, d), (float)softmax_scale, max_query_len, max_seq_len, window,
                                 io_dtype(query), stream_of(kv_cache)),
               op);
  return output;
}

TORCH_LIBRARY_FRAGMENT(custom_esimd_kernels_vllm, m) {
  m.def("esimd_kv_plan(Tensor query_lens, Tensor context_lens, Tensor(a!) block_table, Tensor free_pages, "
        "Tensor free_count, int page_size, Tensor(b!) query_start, Tensor(c!) seq_lens, Tensor(d!) free_count_out, "
        "Tensor(e!) positions, Tensor(f!) slot_mapping) -> Tensor(f!)");
  m.impl("esimd_kv_plan", c10::DispatchKey::CUDA, &esimd_kv_plan);

  m.def("esimd_kv4_append(Tensor key, Tensor value, Tensor kv_scales, Tensor slot_mapping, Tensor(a!) kv_cache, "
        "int page_size) -> Tensor(a!)");
  m.impl("esimd_kv4_append", c10::DispatchKey::CUDA, &esimd_kv4_append);

  m.def("esimd_kv4_gather(Tensor kv_cache, Tensor kv_scales, Tensor slots, Tensor(a!) key, Tensor(b!) value, "
        "int page_size) -> ()");
  m.impl("esimd_kv4_gather", c10::DispatchKey::CUDA, &esimd_kv4_gather);

  m.def("esimd_kv4_attention(Tensor query, Tensor kv_cache, Tensor kv_scales, Tensor block_table, Tensor query_start, "
        "Tensor seq_lens, Tensor(a!) output, int page_size, float softmax_scale, int max_query_len, int max_seq_len, "
        "int window) -> Tensor(a!)");
  m.impl("esimd_kv4_attention", c10::DispatchKey::CUDA, &esimd_kv4_attention);
}

PyMODINIT_FUNC PyInit_custom_esimd_kernels_kv4() {
  static struct PyModuleDef module = {PyModuleDef_HEAD_INIT, "custom_esimd_kernels_kv4", nullptr, 0, nullptr};
  return PyModule_Create(&module);
}
