// Block tables, slot map, positions and lengths of a batch from its request lengths (gfx950).
//
//  bt_requests   one workgroup of 1024 threads.  Each thread owns up to kPerThread consecutive requests; two
//    workgroup scans give the packed token offsets and freed pages, then the wanted pages (what fits depends on
//    the first).  The offsets lie in LDS, and freed pages, fresh pages and (small batches) tokens are each
//    spread over all threads: a thread finds its request by binary search, so one long prompt is as quick as
//    many short ones.  Freed pages are on the stack before any is taken from it: one call does both.
//  bt_tokens     slots and positions of larger batches, a grid of workgroups that hold cu_lens in LDS.
//
// The work is a few bytes a token: what a call costs is its launches and the chain of dependent loads and
// barriers in the first (lengths, two scans, stack, table).

#include "l20_block_tables.h"

#include <algorithm>

#include "l20_latent_common.h"

namespace l20bt {

constexpr int kThreads = 1024;
constexpr int kPerThread = L20_PD_MAX_REQUESTS / kThreads;
// Tokens that bt_requests places itself; more go to bt_tokens in a second launch.
constexpr int kTokensInline = 4096;

struct Params {
  const int32_t *cached, *fresh;
  int32_t *table;
  int64_t t_sr;
  int width;
  int32_t *stack;
  int pool;
  const int32_t *count;
  int32_t *count_out;
  int64_t *slots, *positions;
  int tokens;
  int32_t *cu, *seq_lens;
  int batch, page;
  int inline_tokens;
};

// Inclusive scan of one value a thread over the workgroup; `total` is the sum.
__device__ __forceinline__ int64_t scan(int64_t x, int64_t *s_wave, int64_t &total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const int64_t y = __shfl_up(x, off);
    if (lane >= off) x += y;
  }
  __syncthreads();  // s_wave may still be read from the scan before
  if (lane == 63) s_wave[wave] = x;
  __syncthreads();
  int64_t before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < kThreads / 64; ++w) {
    const int64_t v = s_wave[w];
    before += w < wave ? v : 0;
    total += v;
  }
  return x + before;
}

// The request whose range [at[b], at[b + 1]) holds x (at[0] = 0 <= x < at[n]).
__device__ __forceinline__ int find(const int *at, int n, int x) {
  int lo = 0, hi = n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (at[mid] <= x) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

__device__ __forceinline__ int clamp32(int64_t x) { return (int)(x < INT32_MAX ? x : INT32_MAX); }

__device__ __forceinline__ void place(const Params &p, int t, int start, int cached, bool served, int b) {
  const int64_t pos = (int64_t)cached + (t - start);
  int64_t slot = -1;
  if (served) {  // its pages are inside the table's width
    const int64_t row = pos / p.page;
    const int page = p.table[b * p.t_sr + row];
    if (page >= 0) slot = (int64_t)page * p.page + (pos - row * p.page);
  }
  p.slots[t] = slot;
  p.positions[t] = pos;
}

__global__ __launch_bounds__(kThreads) void bt_requests(Params p) {
  extern __shared__ int s_mem[];
  __shared__ int64_t s_wave[kThreads / 64];
  __shared__ int s_taken;
  int *const s_cu = s_mem;                // [batch + 1] token offsets
  int *const s_back = s_cu + p.batch + 1;  // [batch + 1] freed pages
  int *const s_need = s_back + p.batch + 1;
  int *const s_len = s_need + p.batch + 1;  // cached tokens, -1 - cached where not served
  const int tid = threadIdx.x;
  const int per = (p.batch + kThreads - 1) / kThreads;
  const int count = min(max(*p.count, 0), p.pool);
  int cached[kPerThread], fresh[kPerThread];
  int64_t tokens = 0, back = 0, total;
#pragma unroll
  for (int i = 0; i < kPerThread; ++i) {
    const int b = tid * per + i;
    cached[i] = fresh[i] = 0;
    if (i < per && b < p.batch) {
      cached[i] = max(p.cached[b], 0);
      fresh[i] = p.fresh[b];
      tokens += max(fresh[i], 0);
      if (fresh[i] < 0) back += min((int)(((int64_t)cached[i] + p.page - 1) / p.page), p.width);
    }
  }
  int64_t token_end = scan(tokens, s_wave, total);
  const int64_t all_tokens = total;
  int64_t back_end = scan(back, s_wave, total);
  const int64_t have = min((int64_t)count + total, (int64_t)p.pool);
  // offsets, and what each request wants
  int64_t at = token_end - tokens, bk = back_end - back, need = 0;
  int want[kPerThread];
#pragma unroll
  for (int i = 0; i < kPerThread; ++i) {
    const int b = tid * per + i;
    want[i] = -1;
    if (i < per && b < p.batch) {
      s_cu[b] = clamp32(at);
      s_back[b] = clamp32(bk);
      const int n = max(fresh[i], 0);
      at += n;
      const int64_t held = ((int64_t)cached[i] + p.page - 1) / p.page;
      const int64_t all = ((int64_t)cached[i] + n + p.page - 1) / p.page;
      if (fresh[i] < 0) bk += min(held, (int64_t)p.width);
      else if (all <= p.width && at <= p.tokens && (int64_t)cached[i] + n <= INT32_MAX) want[i] = (int)(all - held);
      need += max(want[i], 0);
    }
  }
  int64_t need_total;
  const int64_t need_end = scan(need, s_wave, need_total);
  if (tid == 0) {
    s_taken = 0;
    s_cu[p.batch] = clamp32(all_tokens);
    s_back[p.batch] = clamp32(total);
    s_need[p.batch] = clamp32(need_total);
    p.cu[p.batch] = (int)min(all_tokens, (int64_t)p.tokens);
  }
  __syncthreads();
  int64_t taken = need_end - need;
  int most = 0;
#pragma unroll
  for (int i = 0; i < kPerThread; ++i) {
    const int b = tid * per + i;
    if (i < per && b < p.batch) {
      s_need[b] = clamp32(taken);
      const int w = max(want[i], 0);
      taken += w;
      const bool served = want[i] == 0 || (want[i] > 0 && taken <= have);
      if (served && w > 0) most = (int)taken;
      s_len[b] = served ? cached[i] : -1 - cached[i];
      p.cu[b] = min(s_cu[b], p.tokens);
      p.seq_lens[b] = served ? cached[i] + fresh[i] : (fresh[i] < 0 ? 0 : cached[i]);
    }
  }
  if (most) atomicMax(&s_taken, most);  // (a maximum has no order)
  // freed pages onto the stack
  const int freed = s_back[p.batch];
  for (int64_t k = tid; k < freed && count + k < p.pool; k += kThreads) {
    const int b = find(s_back, p.batch, (int)k);
    p.stack[count + k] = p.table[b * p.t_sr + ((int)k - s_back[b])];
  }
  __syncthreads();
  // fresh pages from its top
  const int used = s_taken;
  for (int64_t k = tid; k < used; k += kThreads) {
    const int b = find(s_need, p.batch, (int)k);
    const int64_t held = ((int64_t)s_len[b] + p.page - 1) / p.page;  // served: s_len is the cached length
    p.table[b * p.t_sr + held + (k - s_need[b])] = p.stack[have - 1 - k];
  }
  if (tid == 0) *p.count_out = (int)have - used;
  if (!p.inline_tokens) return;
  __syncthreads();
  for (int64_t t = tid; t < p.tokens; t += kThreads) {
    if (t >= all_tokens) {
      p.slots[t] = -1;
      p.positions[t] = 0;
      continue;
    }
    const int b = find(s_cu, p.batch, (int)t);
    const int len = s_len[b];
    place(p, (int)t, s_cu[b], len >= 0 ? len : -1 - len, len >= 0, b);
  }
}

__global__ __launch_bounds__(256) void bt_tokens(Params p, int per_block) {
  extern __shared__ int s_cu[];
  for (int b = threadIdx.x; b <= p.batch; b += 256) s_cu[b] = p.cu[b];
  __syncthreads();
  const int64_t first = (int64_t)blockIdx.x * per_block;
  const int64_t end = min(first + per_block, (int64_t)p.tokens);
  for (int64_t t = first + threadIdx.x; t < end; t += 256) {
    if (t >= s_cu[p.batch]) {
      p.slots[t] = -1;
      p.positions[t] = 0;
      continue;
    }
    const int b = find(s_cu, p.batch, (int)t);
    const int cached = max(p.cached[b], 0);
    // (a request with tokens is served if and only if its length has grown)
    place(p, (int)t, s_cu[b], cached, p.seq_lens[b] != cached, b);
  }
}

}  // namespace l20bt

namespace {

using l20pd_host::set_error;

int32_t check(const l20_pd_block_tables_args *a) {
  if (!a) return set_error(L20_PD_EINVAL, "null argument block");
  if (a->batch < 0 || a->batch > L20_PD_MAX_REQUESTS)
    return set_error(L20_PD_EINVAL, "block tables: at most 8192 requests");
  if (a->page_size < 16 || a->page_size % 16 || a->page_size > 4096)
    return set_error(L20_PD_EINVAL, "page size must be a multiple of 16 up to 4096");
  if ((a->batch > 0 && a->table_pages < 1) || a->pool < 1 || a->num_slots < 0)
    return set_error(L20_PD_EINVAL, "block table and page pool must not be empty");
  if ((a->batch > 0 && (!a->cached_lens || !a->new_lens || !a->block_table || !a->seq_lens)) || !a->free_pages ||
      !a->free_count || !a->free_count_out || !a->cu_lens || (a->num_slots > 0 && (!a->slots || !a->positions)))
    return set_error(L20_PD_EINVAL, "null tensor pointer");
  if (a->batch > 0 && (a->seq_lens == a->cached_lens || a->seq_lens == a->new_lens))
    return set_error(L20_PD_EINVAL, "seq_lens must not be cached_lens or new_lens");
  return L20_PD_OK;
}

int32_t launched() {
  const hipError_t e = hipGetLastError();
  if (e == hipSuccess) return L20_PD_OK;
  char msg[256];
  snprintf(msg, sizeof(msg), "HIP launch failed: %s", hipGetErrorString(e));
  return set_error(L20_PD_ELAUNCH, msg);
}

}  // namespace

extern "C" {

int32_t l20_pd_block_tables_check(const l20_pd_block_tables_args *a) {
  l20pd_host::clear_error();
  return check(a);
}

int32_t l20_pd_block_tables(const l20_pd_block_tables_args *a, void *stream) {
  l20pd_host::clear_error();
  const int32_t rc = check(a);
  if (rc != L20_PD_OK) return rc;
  l20bt::Params p{};
  p.cached = a->cached_lens;
  p.fresh = a->new_lens;
  p.table = a->block_table;
  p.t_sr = a->bt_stride_row;
  p.width = a->table_pages;
  p.stack = a->free_pages;
  p.pool = a->pool;
  p.count = a->free_count;
  p.count_out = a->free_count_out;
  p.slots = a->slots;
  p.positions = a->positions;
  p.tokens = a->num_slots;
  p.cu = a->cu_lens;
  p.seq_lens = a->seq_lens;
  p.batch = a->batch;
  p.page = a->page_size;
  p.inline_tokens = a->num_slots <= l20bt::kTokensInline;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const size_t lds = (size_t)(4 * (a->batch + 1)) * sizeof(int);  // at most 128 KB
  static l20la::LdsLimit limit;
  const hipError_t e = limit.raise(reinterpret_cast<const void *>(&l20bt::bt_requests), 4 * (L20_PD_MAX_REQUESTS + 1) * (int)sizeof(int));
  if (e != hipSuccess) return set_error(L20_PD_ELAUNCH, hipGetErrorString(e));
  hipLaunchKernelGGL(l20bt::bt_requests, dim3(1), dim3(l20bt::kThreads), lds, s, p);
  int32_t r = launched();
  if (r != L20_PD_OK || p.inline_tokens) return r;
  const int per_block = 1024;
  hipLaunchKernelGGL(l20bt::bt_tokens, dim3((unsigned)(((int64_t)p.tokens + per_block - 1) / per_block)), dim3(256),
                     (size_t)(a->batch + 1) * sizeof(int), s, p, per_block);
  return launched();
}

}  // extern "C"
