// TORCH_LIBRARY(l20_stack) binding of latent attention, its cache producer and the block-table builder
// (include/l20_latent_attention.h, include/l20_block_tables.h).  As the paged decode ops: argument checks with
// messages, the C ABI on the current HIP stream of the tensors' device, nothing allocated.

#include <ATen/ATen.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <c10/core/DeviceGuard.h>
#include <torch/library.h>

#include <algorithm>
#include <optional>

#include "l20_block_tables.h"
#include "l20_latent_attention.h"

namespace {

int32_t dtype_code(const at::Tensor &t) {
  return t.scalar_type() == at::kBFloat16 ? L20_PD_BF16 : t.scalar_type() == at::kHalf ? L20_PD_FP16
         : t.scalar_type() == at::kFloat  ? L20_PD_FP32
                                          : -1;
}

int32_t cache_code(const at::Tensor &t) {
  switch (t.scalar_type()) {
    case at::kFloat8_e4m3fn:
      return L20_PD_KV_FP8_E4M3;
    case at::kHalf:
      return L20_PD_KV_FP16;
    case at::kBFloat16:
      return L20_PD_KV_BF16;
    default:
      return -1;
  }
}

void check_device(const at::Tensor &t, const at::Tensor &first) {
  TORCH_CHECK(t.device() == first.device(), "every tensor must be on the same device");
}

int32_t int32(int64_t x, const char *what) {
  TORCH_CHECK(x >= 0 && x <= INT32_MAX, what, " out of range");
  return (int32_t)x;
}

// The stride of a dimension; of one of size 1, whose stride says nothing, what it would be with `inner` per step.
int64_t step(const at::Tensor &t, int64_t dim, int64_t inner) { return t.size(dim) > 1 ? t.stride(dim) : inner; }

void *stream_of(const at::Tensor &t) {
  return at::hip::getCurrentHIPStreamMasqueradingAsCUDA(t.get_device()).stream();
}

void latent_rope_and_cache(const std::optional<at::Tensor> &query, const at::Tensor &latent, const at::Tensor &key_rope,
                           const at::Tensor &positions, const at::Tensor &cos_sin_cache, bool is_neox,
                           const at::Tensor &latent_cache, const at::Tensor &slot_mapping,
                           const std::optional<at::Tensor> &query_out, const at::Tensor &latent_out,
                           const at::Tensor &key_rope_out, const std::optional<at::Tensor> &norm_weight, double norm_eps,
                           double cache_scale) {
  const bool has_q = query.has_value() && query->defined();
  TORCH_CHECK(latent.is_cuda(), "latent must be CUDA");
  TORCH_CHECK(latent.dim() == 2 && latent_out.sizes() == latent.sizes(), "expected latent and latent_out [tokens, rank]");
  const int64_t tokens = latent.size(0), rank = latent.size(1);
  TORCH_CHECK(key_rope.dim() == 2 && key_rope.size(0) == tokens && key_rope_out.sizes() == key_rope.sizes(),
              "expected key_rope and key_rope_out [tokens, rope]");
  TORCH_CHECK(latent_cache.dim() == 3 && latent_cache.size(2) == rank + key_rope.size(1),
              "latent cache must be [pages, page, rank + 64] with rank 256 or 512");
  TORCH_CHECK(positions.scalar_type() == at::kLong && positions.dim() == 1 && positions.is_contiguous() &&
                  positions.size(0) == tokens && slot_mapping.scalar_type() == at::kLong && slot_mapping.dim() == 1 &&
                  slot_mapping.is_contiguous() && slot_mapping.size(0) == tokens,
              "positions and slot_mapping must be contiguous int64 [tokens]");
  TORCH_CHECK(cos_sin_cache.dim() == 2 && cos_sin_cache.size(1) == key_rope.size(1) && cos_sin_cache.stride(1) == 1,
              "cos_sin_cache must be [positions, rope]");
  for (const at::Tensor *t : {&latent_out, &key_rope, &key_rope_out})
    TORCH_CHECK(t->scalar_type() == latent.scalar_type(), "latent, key_rope and their outputs must have one dtype");
  for (const at::Tensor *t : {&latent, &latent_out, &key_rope, &key_rope_out, &latent_cache})
    TORCH_CHECK(t->size(-1) <= 1 || t->stride(-1) == 1, "the last dimension must be contiguous");
  for (const at::Tensor *t : {&latent_out, &key_rope, &key_rope_out, &positions, &cos_sin_cache, &latent_cache, &slot_mapping})
    check_device(*t, latent);
  l20_pd_latent_write_args a{};
  if (has_q) {
    TORCH_CHECK(query_out.has_value() && query_out->defined(), "query needs query_out");
    const at::Tensor &q = *query, &o = *query_out;
    TORCH_CHECK(q.dim() == 3 && q.size(0) == tokens && q.size(2) == key_rope.size(1) && o.sizes() == q.sizes(),
                "expected query and query_out [tokens, heads, rope]");
    TORCH_CHECK(q.scalar_type() == latent.scalar_type() && o.scalar_type() == latent.scalar_type(),
                "query must have the latent's dtype");
    TORCH_CHECK(q.stride(2) == 1 && o.stride(2) == 1, "the last dimension must be contiguous");
    check_device(q, latent);
    check_device(o, latent);
    a.query = q.data_ptr();
    a.q_stride_token = step(q, 0, 0);
    a.q_stride_head = step(q, 1, 0);
    a.query_out = o.data_ptr();
    a.qo_stride_token = step(o, 0, 0);
    a.qo_stride_head = step(o, 1, 0);
    a.num_heads = int32(q.size(1), "head count");
  }
  a.latent = latent.data_ptr();
  a.l_stride_token = step(latent, 0, 0);
  a.latent_out = latent_out.data_ptr();
  a.lo_stride_token = step(latent_out, 0, 0);
  a.key = key_rope.data_ptr();
  a.k_stride_token = step(key_rope, 0, 0);
  a.key_out = key_rope_out.data_ptr();
  a.ko_stride_token = step(key_rope_out, 0, 0);
  a.dtype = dtype_code(latent);
  a.positions = positions.data_ptr<int64_t>();
  a.cos_sin_cache = cos_sin_cache.data_ptr();
  a.cs_stride_position = step(cos_sin_cache, 0, 0);
  a.max_position = cos_sin_cache.size(0);
  a.cs_dtype = dtype_code(cos_sin_cache);
  a.is_neox = is_neox;
  if (norm_weight.has_value() && norm_weight->defined()) {
    TORCH_CHECK(norm_weight->dim() == 1 && norm_weight->size(0) == rank && norm_weight->is_contiguous() &&
                    norm_weight->scalar_type() == latent.scalar_type(),
                "norm_weight must be contiguous [rank] of the latent's dtype");
    check_device(*norm_weight, latent);
    a.norm_weight = norm_weight->data_ptr();
  }
  a.norm_eps = (float)norm_eps;
  a.slot_mapping = slot_mapping.data_ptr<int64_t>();
  a.cache = latent_cache.data_ptr();
  a.c_stride_page = step(latent_cache, 0, latent_cache.size(1) * latent_cache.stride(1));
  a.c_stride_token = latent_cache.stride(1);
  a.num_pages = latent_cache.size(0);
  a.page_size = int32(latent_cache.size(1), "page size");
  a.cache_dtype = cache_code(latent_cache);
  a.cache_scale = (float)cache_scale;
  a.num_tokens = int32(tokens, "token count");
  a.rank = int32(rank, "rank");
  a.rope_dim = int32(key_rope.size(1), "rotary dims");
  const c10::DeviceGuard guard(latent.device());
  TORCH_CHECK(l20_pd_latent_rope_and_cache(&a, stream_of(latent)) == L20_PD_OK, l20_pd_last_error());
}

at::Tensor paged_latent(const at::Tensor &query, const at::Tensor &latent_cache, const at::Tensor &block_table,
                        const at::Tensor &seq_lens, const at::Tensor &output, const std::optional<at::Tensor> &workspace,
                        double softmax_scale, double cache_scale, int64_t max_seq_len, int64_t q_len,
                        const std::optional<at::Tensor> &lse) {
  TORCH_CHECK(query.is_cuda(), "query must be CUDA");
  TORCH_CHECK(query.dim() == 3, "expected query [batch * q_len, heads, rank + rope]");
  TORCH_CHECK(latent_cache.dim() == 3 && latent_cache.size(2) == query.size(2),
              "latent cache must be [pages, page, rank + rope]");
  TORCH_CHECK(q_len >= 1 && query.size(0) % q_len == 0, "query rows must be batch * q_len");
  const int64_t rows = query.size(0), batch = rows / q_len;
  TORCH_CHECK(output.dim() == 3 && output.size(0) == rows && output.size(1) == query.size(1) &&
                  output.size(2) < query.size(2) && output.scalar_type() == query.scalar_type(),
              "output must be [batch * q_len, heads, rank] of the query's dtype");
  TORCH_CHECK(block_table.dim() == 2 && block_table.size(0) == batch && block_table.scalar_type() == at::kInt &&
                  (block_table.size(1) <= 1 || block_table.stride(1) == 1),
              "block table must be int32 [batch, pages] with contiguous rows");
  TORCH_CHECK(seq_lens.dim() == 1 && seq_lens.size(0) == batch && seq_lens.scalar_type() == at::kInt && seq_lens.is_contiguous(),
              "seq_lens must be contiguous int32 [batch]");
  TORCH_CHECK(query.stride(2) == 1 && latent_cache.stride(2) == 1 && output.stride(2) == 1,
              "the last dimension must be contiguous");
  for (const at::Tensor *t : {&latent_cache, &block_table, &seq_lens, &output}) check_device(*t, query);
  l20_pd_latent_args a{};
  if (lse.has_value() && lse->defined()) {
    TORCH_CHECK(lse->scalar_type() == at::kFloat && lse->dim() == 2 && lse->size(0) == rows && lse->size(1) == query.size(1),
                "lse must be fp32 [batch * q_len, heads]");
    check_device(*lse, query);
    a.lse = lse->data_ptr<float>();
    a.lse_stride_row = lse->stride(0);
    a.lse_stride_head = lse->stride(1);
  }
  if (workspace.has_value() && workspace->defined()) {
    TORCH_CHECK(workspace->is_contiguous(), "workspace must be contiguous");
    check_device(*workspace, query);
    a.workspace = workspace->data_ptr();
    a.workspace_bytes = (int64_t)workspace->nbytes();
  }
  a.query = query.data_ptr();
  a.q_stride_row = step(query, 0, 0);
  a.q_stride_head = step(query, 1, 0);
  a.dtype = dtype_code(query);
  a.cache = latent_cache.data_ptr();
  a.c_stride_page = step(latent_cache, 0, latent_cache.size(1) * latent_cache.stride(1));
  a.c_stride_token = latent_cache.stride(1);
  a.num_pages = latent_cache.size(0);
  a.page_size = int32(latent_cache.size(1), "page size");
  a.cache_dtype = cache_code(latent_cache);
  a.cache_scale = (float)cache_scale;
  a.block_table = block_table.data_ptr<int32_t>();
  a.bt_stride_row = step(block_table, 0, block_table.size(1));
  a.table_pages = int32(block_table.size(1), "block table width");
  a.seq_lens = seq_lens.data_ptr<int32_t>();
  a.output = output.data_ptr();
  a.o_stride_row = step(output, 0, 0);
  a.o_stride_head = step(output, 1, 0);
  a.softmax_scale = (float)softmax_scale;
  a.batch = int32(batch, "batch");
  a.q_len = int32(q_len, "q_len");
  a.num_heads = int32(query.size(1), "head count");
  a.rank = int32(output.size(2), "rank");
  a.rope_dim = int32(query.size(2) - output.size(2), "rotary dims");
  a.max_seq_len = int32(max_seq_len, "max_seq_len");
  const c10::DeviceGuard guard(query.device());
  TORCH_CHECK(l20_pd_paged_latent(&a, stream_of(query)) == L20_PD_OK, l20_pd_last_error());
  return output;
}

at::Tensor latent_prompt(const at::Tensor &query, const at::Tensor &key, const at::Tensor &key_rope, const at::Tensor &value,
                         const at::Tensor &cu_seqlens_q, const at::Tensor &cu_seqlens_k, int64_t max_seqlen_q,
                         const at::Tensor &output, double softmax_scale, bool causal, const std::optional<at::Tensor> &lse,
                         const std::optional<at::Tensor> &workspace) {
  TORCH_CHECK(query.is_cuda(), "query must be CUDA");
  TORCH_CHECK(query.dim() == 3 && key.dim() == 3 && value.dim() == 3 && key_rope.dim() == 2 && output.dim() == 3,
              "expected query, key, value and output [tokens, heads, dims] and key_rope [tokens, rope]");
  TORCH_CHECK(key.size(0) == value.size(0) && key.size(0) == key_rope.size(0) && key.size(1) == query.size(1) &&
                  value.size(1) == query.size(1),
              "keys and values must have the same tokens, and the query's heads");
  TORCH_CHECK(query.size(2) == key.size(2) + key_rope.size(1), "query dims must be the key's and key_rope's");
  TORCH_CHECK(output.size(0) == query.size(0) && output.size(1) == query.size(1) && output.size(2) == value.size(2),
              "output must be [tokens, heads, value dims]");
  for (const at::Tensor *t : {&key, &key_rope, &value, &output})
    TORCH_CHECK(t->scalar_type() == query.scalar_type(), "query, keys, values and output must have one dtype");
  TORCH_CHECK(cu_seqlens_q.dim() == 1 && cu_seqlens_q.size(0) >= 1 && cu_seqlens_k.sizes() == cu_seqlens_q.sizes() &&
                  cu_seqlens_q.scalar_type() == at::kInt && cu_seqlens_k.scalar_type() == at::kInt &&
                  cu_seqlens_q.is_contiguous() && cu_seqlens_k.is_contiguous(),
              "cu_seqlens must be contiguous int32 [batch + 1]");
  for (const at::Tensor *t : {&query, &key, &key_rope, &value, &output})
    TORCH_CHECK(t->stride(-1) == 1, "the last dimension must be contiguous");
  for (const at::Tensor *t : {&key, &key_rope, &value, &cu_seqlens_q, &cu_seqlens_k, &output}) check_device(*t, query);
  l20_pd_latent_prompt_args a{};
  if (lse.has_value() && lse->defined()) {
    TORCH_CHECK(lse->scalar_type() == at::kFloat && lse->dim() == 2 && lse->size(0) == query.size(0) &&
                    lse->size(1) == query.size(1),
                "lse must be fp32 [tokens, heads]");
    check_device(*lse, query);
    a.lse = lse->data_ptr<float>();
    a.lse_stride_token = lse->stride(0);
    a.lse_stride_head = lse->stride(1);
  }
  if (workspace.has_value() && workspace->defined() && workspace->nbytes() > 0) {
    TORCH_CHECK(workspace->is_contiguous(), "workspace must be contiguous");
    check_device(*workspace, query);
    a.workspace = workspace->data_ptr();
    a.workspace_bytes = (int64_t)workspace->nbytes();
  }
  a.query = query.data_ptr();
  a.q_stride_token = step(query, 0, 0);
  a.q_stride_head = step(query, 1, 0);
  a.key = key.data_ptr();
  a.k_stride_token = step(key, 0, 0);
  a.k_stride_head = step(key, 1, 0);
  a.key_rope = key_rope.data_ptr();
  a.kr_stride_token = step(key_rope, 0, 0);
  a.value = value.data_ptr();
  a.v_stride_token = step(value, 0, 0);
  a.v_stride_head = step(value, 1, 0);
  a.dtype = dtype_code(query);
  a.cu_q = cu_seqlens_q.data_ptr<int32_t>();
  a.cu_k = cu_seqlens_k.data_ptr<int32_t>();
  a.output = output.data_ptr();
  a.o_stride_token = step(output, 0, 0);
  a.o_stride_head = step(output, 1, 0);
  a.softmax_scale = (float)softmax_scale;
  a.causal = causal;
  a.total_q = query.size(0);
  a.total_k = key.size(0);
  a.batch = int32(cu_seqlens_q.size(0) - 1, "batch");
  a.num_heads = int32(query.size(1), "head count");
  a.max_q_len = int32(max_seqlen_q, "max_seqlen_q");
  a.head_dim = int32(key.size(2), "key dims");
  a.rope_dim = int32(key_rope.size(1), "rotary dims");
  a.value_dim = int32(value.size(2), "value dims");
  const c10::DeviceGuard guard(query.device());
  TORCH_CHECK(l20_pd_latent_prompt(&a, stream_of(query)) == L20_PD_OK, l20_pd_last_error());
  return output;
}

void build_block_tables(const at::Tensor &cached_lens, const at::Tensor &new_lens, const at::Tensor &block_table,
                        const at::Tensor &free_pages, const at::Tensor &free_count, const at::Tensor &slot_mapping,
                        const at::Tensor &positions, const at::Tensor &cu_lens, const at::Tensor &seq_lens, int64_t page_size,
                        const at::Tensor &free_count_out) {
  TORCH_CHECK(block_table.is_cuda(), "block_table must be CUDA");
  TORCH_CHECK(cached_lens.dim() == 1, "cached_lens must be [requests]");
  const int64_t batch = cached_lens.size(0);
  for (const at::Tensor *t : {&cached_lens, &new_lens, &seq_lens})
    TORCH_CHECK(t->scalar_type() == at::kInt && t->dim() == 1 && t->size(0) == batch && t->is_contiguous(),
                "cached_lens, new_lens and seq_lens must be contiguous int32 [requests]");
  TORCH_CHECK(block_table.scalar_type() == at::kInt && block_table.dim() == 2 && block_table.size(0) == batch &&
                  (block_table.size(1) <= 1 || block_table.stride(1) == 1),
              "block table must be int32 [requests, pages] with contiguous rows");
  TORCH_CHECK(free_pages.scalar_type() == at::kInt && free_pages.dim() == 1 && free_pages.is_contiguous(),
              "free_pages must be contiguous int32 [pool]");
  for (const at::Tensor *t : {&free_count, &free_count_out})
    TORCH_CHECK(t->scalar_type() == at::kInt && t->numel() == 1, "free_count must be one int32");
  TORCH_CHECK(slot_mapping.scalar_type() == at::kLong && slot_mapping.dim() == 1 && slot_mapping.is_contiguous() &&
                  positions.scalar_type() == at::kLong && positions.sizes() == slot_mapping.sizes() && positions.is_contiguous(),
              "slot_mapping and positions must be contiguous int64 [tokens]");
  TORCH_CHECK(cu_lens.scalar_type() == at::kInt && cu_lens.dim() == 1 && cu_lens.size(0) == batch + 1 && cu_lens.is_contiguous(),
              "cu_seqlens must be contiguous int32 [requests + 1]");
  for (const at::Tensor *t : {&cached_lens, &new_lens, &free_pages, &free_count, &free_count_out, &slot_mapping, &positions,
                              &cu_lens, &seq_lens})
    check_device(*t, block_table);
  l20_pd_block_tables_args a{};
  a.cached_lens = cached_lens.data_ptr<int32_t>();
  a.new_lens = new_lens.data_ptr<int32_t>();
  a.block_table = block_table.data_ptr<int32_t>();
  a.bt_stride_row = step(block_table, 0, block_table.size(1));
  a.table_pages = int32(block_table.size(1), "block table width");
  a.free_pages = free_pages.data_ptr<int32_t>();
  a.pool = int32(free_pages.size(0), "page pool");
  a.free_count = free_count.data_ptr<int32_t>();
  a.free_count_out = free_count_out.data_ptr<int32_t>();
  a.slots = slot_mapping.data_ptr<int64_t>();
  a.positions = positions.data_ptr<int64_t>();
  a.num_slots = int32(slot_mapping.size(0), "token count");
  a.cu_lens = cu_lens.data_ptr<int32_t>();
  a.seq_lens = seq_lens.data_ptr<int32_t>();
  a.batch = int32(batch, "request count");
  a.page_size = int32(page_size, "page size");
  const c10::DeviceGuard guard(block_table.device());
  TORCH_CHECK(l20_pd_block_tables(&a, stream_of(block_table)) == L20_PD_OK, l20_pd_last_error());
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(l20_stack, m) {
  m.def(
      "latent_rope_and_cache(Tensor? query, Tensor latent, Tensor key_rope, Tensor positions, "
      "Tensor cos_sin_cache, bool is_neox, Tensor(a!) latent_cache, Tensor slot_mapping, "
      "Tensor(b!)? query_out, Tensor(c!) latent_out, Tensor(d!) key_rope_out, "
      "Tensor? norm_weight=None, float norm_eps=1e-6, float cache_scale=1.0) -> ()");
  m.def(
      "paged_latent_attention_out(Tensor query, Tensor latent_cache, Tensor block_table, Tensor seq_lens, "
      "Tensor(a!) output, Tensor(b!)? workspace, float softmax_scale, float cache_scale, int max_seq_len, "
      "int q_len=1, Tensor(c!)? lse=None) -> Tensor(a!)");
  m.def(
      "latent_prompt_attention_out(Tensor query, Tensor key, Tensor key_rope, Tensor value, "
      "Tensor cu_seqlens_q, Tensor cu_seqlens_k, int max_seqlen_q, Tensor(a!) output, float softmax_scale, "
      "bool causal=True, Tensor(b!)? lse=None, Tensor(c!)? workspace=None) -> Tensor(a!)");
  m.def(
      "build_block_tables(Tensor cached_lens, Tensor new_lens, Tensor(a!) block_table, Tensor(b!) free_pages, "
      "Tensor free_count, Tensor(c!) slot_mapping, Tensor(d!) positions, Tensor(e!) cu_seqlens, "
      "Tensor(f!) seq_lens, int page_size, Tensor(g!) free_count_out) -> ()");
}

TORCH_LIBRARY_IMPL(l20_stack, CUDA, m) {
  m.impl("latent_rope_and_cache", &latent_rope_and_cache);
  m.impl("paged_latent_attention_out", &paged_latent);
  m.impl("latent_prompt_attention_out", &latent_prompt);
  m.impl("build_block_tables", &build_block_tables);
}
