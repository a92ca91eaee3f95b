// TORCH_LIBRARY(l20_stack) binding of beam search's selection and of the page pool's operators
// (include/l20_beam_search.h, include/l20_block_tables.h).  As the other ops: argument checks with messages, the C
// ABI on the current HIP stream of the tensors' device, nothing allocated.

#include <ATen/ATen.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <c10/core/DeviceGuard.h>
#include <torch/library.h>

#include <algorithm>
#include <array>
#include <optional>
#include <vector>

#include "l20_beam_search.h"
#include "l20_block_tables.h"

namespace {

void check_device(const at::Tensor &t, const at::Tensor &first) {
  TORCH_CHECK(t.device() == first.device(), "every tensor must be on the same device");
}

int32_t int32(int64_t x, const char *what) {
  TORCH_CHECK(x >= INT32_MIN && x <= INT32_MAX, what, " out of range");
  return (int32_t)x;
}

// The stride of a dimension; of one of size 1, whose stride says nothing, what it would be with `inner` per step.
int64_t step(const at::Tensor &t, int64_t dim, int64_t inner) { return t.size(dim) > 1 ? t.stride(dim) : inner; }

void *stream_of(const at::Tensor &t) {
  return at::hip::getCurrentHIPStreamMasqueradingAsCUDA(t.get_device()).stream();
}

bool vector_of(const at::Tensor &t, at::ScalarType type, int64_t size) {
  return t.scalar_type() == type && t.dim() == 1 && t.size(0) == size && t.is_contiguous();
}

void beam_search_step(const at::Tensor &logits, const at::Tensor &scores, at::IntArrayRef end_tokens, const at::Tensor &tokens,
                      const at::Tensor &parents, const at::Tensor &scores_out, const at::Tensor &ended_tokens,
                      const at::Tensor &ended_parents, const at::Tensor &ended_scores, const at::Tensor &workspace) {
  TORCH_CHECK(logits.is_cuda(), "logits must be CUDA");
  TORCH_CHECK(scores.dim() == 2 && scores.scalar_type() == at::kFloat, "scores must be fp32 [requests, beams]");
  const int64_t requests = scores.size(0), beams = scores.size(1);
  TORCH_CHECK((logits.dim() == 2 && logits.size(0) == requests * beams) ||
                  (logits.dim() == 3 && logits.size(0) == requests && logits.size(1) == beams),
              "logits must be [requests * beams, vocab] or [requests, beams, vocab]");
  TORCH_CHECK(logits.size(-1) <= 1 || logits.stride(-1) == 1, "the last dimension must be contiguous");
  const at::ScalarType type = logits.scalar_type();
  TORCH_CHECK(type == at::kBFloat16 || type == at::kHalf || type == at::kFloat, "logits must be bf16, fp16 or fp32");
  for (const at::Tensor *t : {&tokens, &ended_tokens})
    TORCH_CHECK(t->scalar_type() == at::kLong && t->sizes() == scores.sizes() && t->is_contiguous(),
                "tokens must be contiguous int64 [requests, beams]");
  for (const at::Tensor *t : {&parents, &ended_parents})
    TORCH_CHECK(t->scalar_type() == at::kInt && t->sizes() == scores.sizes() && t->is_contiguous(),
                "parents must be contiguous int32 [requests, beams]");
  for (const at::Tensor *t : {&scores_out, &ended_scores})
    TORCH_CHECK(t->scalar_type() == at::kFloat && t->sizes() == scores.sizes() && t->is_contiguous(),
                "scores must be contiguous fp32 [requests, beams]");
  TORCH_CHECK(workspace.is_contiguous(), "workspace must be contiguous");
  for (const at::Tensor *t : {&scores, &tokens, &parents, &scores_out, &ended_tokens, &ended_parents, &ended_scores, &workspace})
    check_device(*t, logits);
  TORCH_CHECK(end_tokens.size() <= L20_PD_MAX_END_TOKENS, "at most 8 end tokens");
  int32_t ends[L20_PD_MAX_END_TOKENS];
  for (size_t i = 0; i < end_tokens.size(); ++i) ends[i] = int32(end_tokens[i], "end token");
  l20_pd_beam_step_args a{};
  a.logits = logits.data_ptr();
  if (logits.dim() == 3) {
    a.l_stride_request = step(logits, 0, 0);
    a.l_stride_beam = step(logits, 1, 0);
  } else {
    a.l_stride_beam = step(logits, 0, 0);
    a.l_stride_request = beams * a.l_stride_beam;
  }
  a.dtype = type == at::kBFloat16 ? L20_PD_BF16 : type == at::kHalf ? L20_PD_FP16 : L20_PD_FP32;
  a.scores = scores.data_ptr<float>();
  a.s_stride_request = step(scores, 0, beams);
  a.s_stride_beam = step(scores, 1, 1);
  a.requests = int32(requests, "requests");
  a.beams = int32(beams, "beams");
  a.vocab = int32(logits.size(-1), "vocabulary");
  a.end_tokens = ends;
  a.num_end_tokens = (int32_t)end_tokens.size();
  a.tokens = tokens.data_ptr<int64_t>();
  a.parents = parents.data_ptr<int32_t>();
  a.scores_out = scores_out.data_ptr<float>();
  a.ended_tokens = ended_tokens.data_ptr<int64_t>();
  a.ended_parents = ended_parents.data_ptr<int32_t>();
  a.ended_scores = ended_scores.data_ptr<float>();
  a.workspace = workspace.data_ptr();
  a.workspace_bytes = (int64_t)workspace.nbytes();
  const c10::DeviceGuard guard(logits.device());
  TORCH_CHECK(l20_pd_beam_step(&a, stream_of(logits)) == L20_PD_OK, l20_pd_last_error());
}

// What reorder_block_tables and compact_pages have in common.
template <typename A>
void pool_args(A &a, const at::Tensor &block_table, const at::Tensor &seq_lens, const at::Tensor &page_shares,
               const at::Tensor &free_pages, const at::Tensor &free_count, int64_t page_size, const at::Tensor &src,
               const at::Tensor &dst, const at::Tensor &tokens, const at::Tensor &count, const at::Tensor &workspace) {
  TORCH_CHECK(block_table.is_cuda(), "block_table must be CUDA");
  TORCH_CHECK(block_table.scalar_type() == at::kInt && block_table.dim() == 2 &&
                  (block_table.size(1) <= 1 || block_table.stride(1) == 1),
              "block table must be int32 [rows, pages] with contiguous rows");
  TORCH_CHECK(vector_of(seq_lens, at::kInt, block_table.size(0)), "seq_lens must be contiguous int32 [rows]");
  TORCH_CHECK(page_shares.dim() == 1 && vector_of(page_shares, at::kInt, page_shares.size(0)),
              "page_shares must be contiguous int32 [pages]");
  TORCH_CHECK(free_pages.dim() == 1 && vector_of(free_pages, at::kInt, free_pages.size(0)),
              "free_pages must be contiguous int32 [pool]");
  TORCH_CHECK(free_count.scalar_type() == at::kInt && free_count.numel() == 1, "free_count must be one int32");
  TORCH_CHECK(src.dim() == 1 && vector_of(src, at::kInt, src.size(0)) && vector_of(dst, at::kInt, src.size(0)) &&
                  vector_of(tokens, at::kInt, src.size(0)) && vector_of(count, at::kInt, 2),
              "copies must be contiguous int32: src, dst and tokens [room], count [2]");
  TORCH_CHECK(workspace.is_contiguous(), "workspace must be contiguous");
  const at::Tensor *const all[] = {&block_table, &seq_lens, &page_shares, &free_pages, &free_count,
                                   &src,         &dst,      &tokens,      &count,      &workspace};
  for (const at::Tensor *t : all) check_device(*t, block_table);
  a.block_table = block_table.data_ptr<int32_t>();
  a.bt_stride_row = step(block_table, 0, block_table.size(1));
  a.table_pages = int32(block_table.size(1), "block table width");
  a.seq_lens = seq_lens.data_ptr<int32_t>();
  a.page_shares = page_shares.data_ptr<int32_t>();
  a.pages = int32(page_shares.size(0), "pages");
  a.free_pages = free_pages.data_ptr<int32_t>();
  a.pool = int32(free_pages.size(0), "page pool");
  a.free_count = free_count.data_ptr<int32_t>();
  a.src = src.data_ptr<int32_t>();
  a.dst = dst.data_ptr<int32_t>();
  a.tokens = tokens.data_ptr<int32_t>();
  a.room = int32(src.size(0), "room");
  a.count = count.data_ptr<int32_t>();
  a.page_size = int32(page_size, "page size");
  a.workspace = workspace.data_ptr();
  a.workspace_bytes = (int64_t)workspace.nbytes();
}

void reorder_block_tables(const at::Tensor &parents, const at::Tensor &block_table, const at::Tensor &seq_lens,
                          const at::Tensor &page_shares, const at::Tensor &free_pages, const at::Tensor &free_count,
                          int64_t page_size, const at::Tensor &src, const at::Tensor &dst, const at::Tensor &tokens,
                          const at::Tensor &count, const at::Tensor &workspace) {
  l20_pd_reorder_args a{};
  pool_args(a, block_table, seq_lens, page_shares, free_pages, free_count, page_size, src, dst, tokens, count, workspace);
  TORCH_CHECK(parents.scalar_type() == at::kInt && parents.dim() == 2 && parents.is_contiguous() &&
                  parents.numel() == block_table.size(0),
              "parents must be contiguous int32 [groups, beams], a row of the block table each");
  check_device(parents, block_table);
  a.parents = parents.data_ptr<int32_t>();
  a.groups = int32(parents.size(0), "groups");
  a.beams = int32(parents.size(1), "beams");
  const c10::DeviceGuard guard(block_table.device());
  TORCH_CHECK(l20_pd_reorder_tables(&a, stream_of(block_table)) == L20_PD_OK, l20_pd_last_error());
}

void compact_pages(int64_t limit, const at::Tensor &block_table, const at::Tensor &seq_lens, const at::Tensor &page_shares,
                   const at::Tensor &free_pages, const at::Tensor &free_count, int64_t page_size, const at::Tensor &src,
                   const at::Tensor &dst, const at::Tensor &tokens, const at::Tensor &count, const at::Tensor &workspace) {
  l20_pd_compact_args a{};
  pool_args(a, block_table, seq_lens, page_shares, free_pages, free_count, page_size, src, dst, tokens, count, workspace);
  a.limit = int32(limit, "limit");
  a.rows = int32(block_table.size(0), "rows");
  const c10::DeviceGuard guard(block_table.device());
  TORCH_CHECK(l20_pd_compact_pages(&a, stream_of(block_table)) == L20_PD_OK, l20_pd_last_error());
}

// A cache's layout as the C ABI takes it: [pages, tokens, ...] of any order of dimensions inside a page.
void layout_of(const at::Tensor &cache, bool by_tokens, l20_pd_copy_args &a) {
  struct Dim {
    int64_t size, stride;
    bool token;
  };
  const int64_t item = cache.element_size();
  std::vector<Dim> dims;
  for (int64_t d = 1; d < cache.dim(); ++d)
    if (cache.size(d) != 1) dims.push_back({cache.size(d), cache.stride(d) * item, by_tokens && d == 1});
  std::sort(dims.begin(), dims.end(), [](const Dim &x, const Dim &y) { return x.stride > y.stride; });
  a.inner = item;
  while (!dims.empty() && !dims.back().token && dims.back().stride == a.inner) {
    a.inner *= dims.back().size;
    dims.pop_back();
  }
  for (size_t i = 1; i < dims.size();) {
    Dim &out = dims[i - 1];
    const Dim &in = dims[i];
    if (!out.token && !in.token && out.stride == in.size * in.stride) {
      out = {out.size * in.size, in.stride, false};
      dims.erase(dims.begin() + i);
    } else {
      ++i;
    }
  }
  if (by_tokens && cache.size(1) == 1) dims.insert(dims.begin(), {1, 0, true});
  TORCH_CHECK(dims.size() <= 3, "a page of a cache has too many strides");
  a.pages = cache.size(0);
  a.stride_page = step(cache, 0, 0) * item;
  a.size0 = a.size1 = a.size2 = 1;
  a.stride0 = a.stride1 = a.stride2 = 0;
  a.token_level = -1;
  int64_t *const sizes[3] = {&a.size0, &a.size1, &a.size2}, *const strides[3] = {&a.stride0, &a.stride1, &a.stride2};
  for (size_t i = 0; i < dims.size(); ++i) {
    *sizes[i] = dims[i].size;
    *strides[i] = dims[i].stride;
    if (dims[i].token) a.token_level = (int32_t)i;
  }
}

void copy_pages(const at::Tensor &src, const at::Tensor &dst, const std::optional<at::Tensor> &tokens,
                const std::optional<at::Tensor> &count, at::TensorList caches) {
  TORCH_CHECK(src.is_cuda(), "src must be CUDA");
  TORCH_CHECK(src.dim() == 1 && vector_of(src, at::kInt, src.size(0)) && vector_of(dst, at::kInt, src.size(0)),
              "src and dst must be contiguous int32 [room]");
  check_device(dst, src);
  const bool by_tokens = tokens.has_value() && tokens->defined(), counted = count.has_value() && count->defined();
  if (by_tokens) {
    TORCH_CHECK(vector_of(*tokens, at::kInt, src.size(0)), "tokens must be contiguous int32 [room]");
    check_device(*tokens, src);
  }
  if (counted) {
    TORCH_CHECK(count->scalar_type() == at::kInt && count->dim() == 1 && count->size(0) >= 1 && count->is_contiguous(),
                "count must be contiguous int32");
    check_device(*count, src);
  }
  const c10::DeviceGuard guard(src.device());
  std::vector<void *> same;
  same.reserve(caches.size());
  for (size_t i = 0; i < caches.size();) {  // caches of one layout together
    const at::Tensor &first = caches[i];
    TORCH_CHECK(first.dim() >= 2, "a cache must be [pages, page, ...]");
    TORCH_CHECK(first.numel() > 0, "cache must not be empty");
    same.clear();
    for (; i < caches.size(); ++i) {
      const at::Tensor &cache = caches[i];
      if (cache.element_size() != first.element_size() || cache.sizes() != first.sizes() || cache.strides() != first.strides()) break;
      check_device(cache, src);
      same.push_back(cache.data_ptr());
    }
    l20_pd_copy_args a{};
    layout_of(first, by_tokens, a);
    a.src = src.data_ptr<int32_t>();
    a.dst = dst.data_ptr<int32_t>();
    a.tokens = by_tokens ? tokens->data_ptr<int32_t>() : nullptr;
    a.room = int32(src.size(0), "room");
    a.count = counted ? count->data_ptr<int32_t>() : nullptr;
    a.caches = same.data();
    a.num_caches = int32((int64_t)same.size(), "caches");
    TORCH_CHECK(l20_pd_copy_pages(&a, stream_of(src)) == L20_PD_OK, l20_pd_last_error());
  }
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(l20_stack, m) {
  m.def(
      "beam_search_step(Tensor logits, Tensor scores, int[] end_tokens, Tensor(a!) tokens, Tensor(b!) parents, "
      "Tensor(c!) scores_out, Tensor(d!) ended_tokens, Tensor(e!) ended_parents, Tensor(f!) ended_scores, "
      "Tensor(g!) workspace) -> ()");
  m.def(
      "reorder_block_tables(Tensor parents, Tensor(a!) block_table, Tensor(b!) seq_lens, Tensor(c!) page_shares, "
      "Tensor(d!) free_pages, Tensor(e!) free_count, int page_size, Tensor(f!) src, Tensor(g!) dst, "
      "Tensor(h!) tokens, Tensor(i!) count, Tensor(j!) workspace) -> ()");
  m.def(
      "compact_pages(int limit, Tensor(a!) block_table, Tensor seq_lens, Tensor(b!) page_shares, "
      "Tensor(c!) free_pages, Tensor(d!) free_count, int page_size, Tensor(e!) src, Tensor(f!) dst, "
      "Tensor(g!) tokens, Tensor(h!) count, Tensor(i!) workspace) -> ()");
  m.def("copy_pages(Tensor src, Tensor dst, Tensor? tokens, Tensor? count, Tensor(a!)[] caches) -> ()");
}

TORCH_LIBRARY_IMPL(l20_stack, CUDA, m) {
  m.impl("beam_search_step", &beam_search_step);
  m.impl("reorder_block_tables", &reorder_block_tables);
  m.impl("compact_pages", &compact_pages);
  m.impl("copy_pages", &copy_pages);
}
