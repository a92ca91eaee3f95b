// Block tables, slot map, positions and lengths of a batch from its request lengths (gfx950).
//
//  bt_requests   one workgroup of 1024 threads.  Each thread owns up to kPerThread consecutive requests; two
//    workgroup scans give the packed token offsets and freed pages, then the wanted pages (what fits depends on
//    the first).  The offsets lie in LDS, and freed pages, fresh pages and (small batches) tokens are each
//    spread over all threads: a thread finds its request by binary search, so one long prompt is as quick as
//    many short ones.  Freed pages are on the stack before any is taken from it: one call does both.
//  bt_tokens     slots and positions of larger batches, a token a thread, cu_lens in LDS.
//
// The work is a few bytes a token: what a call costs is its launches (two 3 us apart) and the chain of dependent
// loads and barriers in the first: lengths, two scans, then the stack and the table at once.  256 requests of one
// token take 6.3 us, 48 requests with 20 000 new tokens 10.5 (the empty launch of such a workgroup: 2 to 3); a
// workgroup of 256 threads instead took 7.9, tokens that wait for the table to be written 7.2.

#include "l20_block_tables.h"

#include <algorithm>

#include "l20_latent_common.h"

namespace l20bt {

constexpr int kThreads = 1024;
constexpr int kPerThread = L20_PD_MAX_REQUESTS / kThreads;
// Tokens that bt_requests places itself; more go to bt_tokens in a second launch.  Measured, 256 requests, one launch
// against two: 2048 tokens 7.4 and 8.7 us, 4096 tokens 11.3 and 11.2, 8192 tokens 15.6 and 11.4.
constexpr int kTokensInline = 4096;

// n / page without a division (a good hundred instructions at 64 bits, some thirty at 32), for n through
// 2^31 + 4094, the largest length rounded up by the largest page: n / 16 is below 2^27 + 256 and the magic at most
// 2^36, so their product is below 2^64, and the magic's rounding, below page / 16 <= 2^8, adds less than one step.
constexpr uint64_t page_magic(uint32_t page) { return (((uint64_t)1 << 36) + page / 16 - 1) / (page / 16); }
__host__ __device__ constexpr uint32_t div_magic(uint32_t n, uint64_t magic) { return (uint32_t)((uint64_t)(n >> 4) * magic >> 36); }
// The ends of the first, a middle and the last multiples of every page size.
constexpr bool divides_right() {
  for (uint32_t page = 16; page <= 4096; page += 16)
    for (uint32_t top : {page, (uint32_t)1 << 30, ((uint32_t)1 << 30) + page, (uint32_t)INT32_MAX, (uint32_t)INT32_MAX + page - 1}) {
      const uint32_t at = top / page * page;
      for (uint32_t n : {at - 1, at, at + 1, top})
        if (div_magic(n, page_magic(page)) != n / page) return false;
    }
  return true;
}
static_assert(divides_right(), "the division by the page size");

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
  uint64_t magic;  // division by the page size
  int inline_tokens;
};

__device__ __forceinline__ uint32_t div_page(const Params &p, uint32_t n) { return div_magic(n, p.magic); }
// The pages of n tokens.
__device__ __forceinline__ int pages_of(const Params &p, int n) { return (int)div_page(p, (uint32_t)n + (uint32_t)p.page - 1); }

// Inclusive scans of N values a thread over the workgroup; `total` are the sums.
template <int N> __device__ __forceinline__ void scan(int64_t (&x)[N], int64_t (*s_wave)[kThreads / 64], int64_t (&total)[N]) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1)
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const int64_t y = __shfl_up(x[n], off);
      if (lane >= off) x[n] += y;
    }
#pragma unroll
  for (int n = 0; n < N; ++n)
    if (lane == 63) s_wave[n][wave] = x[n];
  __syncthreads();
#pragma unroll
  for (int n = 0; n < N; ++n) {
    total[n] = 0;
#pragma unroll
    for (int w = 0; w < kThreads / 64; ++w) {
      const int64_t v = s_wave[n][w];
      x[n] += w < wave ? v : 0;
      total[n] += v;
    }
  }
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

__global__ __launch_bounds__(kThreads) void bt_requests(Params p) {
  extern __shared__ int s_mem[];
  __shared__ int64_t s_wave[3][kThreads / 64];
  __shared__ int s_taken;
  int *const s_cu = s_mem;                // [batch + 1] token offsets
  int *const s_back = s_cu + p.batch + 1;  // [batch + 1] freed pages
  int *const s_need = s_back + p.batch + 1;
  int *const s_len = s_need + p.batch + 1;  // cached tokens, -1 - cached where not served
  const int tid = threadIdx.x;
  if (tid == 0) s_taken = 0;
  const int per = (p.batch + kThreads - 1) / kThreads;
  const int count = min(max(*p.count, 0), p.pool);
  int cached[kPerThread], fresh[kPerThread];
  int64_t tokens = 0, back = 0;
#pragma unroll
  for (int i = 0; i < kPerThread; ++i) {
    const int b = tid * per + i;
    cached[i] = fresh[i] = 0;
    if (i < per && b < p.batch) {
      cached[i] = max(p.cached[b], 0);
      fresh[i] = p.fresh[b];
      tokens += max(fresh[i], 0);
      if (fresh[i] < 0) back += min(pages_of(p, cached[i]), p.width);
    }
  }
  int64_t ends[2] = {tokens, back}, totals[2];
  scan<2>(ends, s_wave, totals);
  const int64_t all_tokens = totals[0];
  const int64_t have = min((int64_t)count + totals[1], (int64_t)p.pool);
  // offsets, and what each request wants
  int64_t at = ends[0] - tokens, bk = ends[1] - back, need = 0;
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
      const int held = pages_of(p, cached[i]), all = pages_of(p, (int)min((int64_t)cached[i] + n, (int64_t)INT32_MAX));
      if (fresh[i] < 0) bk += min(held, p.width);
      else if (all <= p.width && at <= p.tokens && (int64_t)cached[i] + n <= INT32_MAX) want[i] = all - held;
      need += max(want[i], 0);
    }
  }
  int64_t need_end[1] = {need}, need_total[1];
  scan<1>(need_end, s_wave + 2, need_total);
  if (tid == 0) {
    s_cu[p.batch] = clamp32(all_tokens);
    s_back[p.batch] = clamp32(totals[1]);
    s_need[p.batch] = clamp32(need_total[0]);
    p.cu[p.batch] = (int)min(all_tokens, (int64_t)p.tokens);
  }
  int64_t taken = need_end[0] - need;
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
  __syncthreads();
  // freed pages onto the stack
  const int freed = s_back[p.batch];
  for (int64_t k = tid; k < freed && count + k < p.pool; k += kThreads) {
    const int b = find(s_back, p.batch, (int)k);
    p.stack[count + k] = p.table[b * p.t_sr + ((int)k - s_back[b])];
  }
  if (freed) __syncthreads();
  // fresh pages from its top; where both are few one half of the workgroup does them and the other the tokens, at the
  // same time (256 requests of one token 6.8 -> 6.3 us)
  const int used = s_taken;
  const bool halves = p.inline_tokens && max(used, p.tokens) <= kThreads / 2;
  for (int64_t k = halves && tid >= kThreads / 2 ? used : tid; k < used; k += kThreads) {
    const int b = find(s_need, p.batch, (int)k);
    const int64_t held = pages_of(p, s_len[b]);  // served: s_len is the cached length
    p.table[b * p.t_sr + held + (k - s_need[b])] = p.stack[have - 1 - k];
  }
  if (tid == 0) *p.count_out = (int)have - used;
  if (!p.inline_tokens) return;
  // (a token's page is one that the request held, or comes from the stack as above: no wait for the table)
  for (int64_t t = !halves ? tid : tid >= kThreads / 2 ? tid - kThreads / 2 : p.tokens; t < p.tokens; t += kThreads) {
    int64_t slot = -1, pos = 0;
    if (t < all_tokens) {
      const int b = find(s_cu, p.batch, (int)t), len = s_len[b];
      const int64_t cached = len >= 0 ? len : -1 - len;
      pos = cached + (t - s_cu[b]);
      if (len >= 0) {
        const int64_t row = div_page(p, (uint32_t)pos), held = pages_of(p, len);
        const int page = row < held ? p.table[b * p.t_sr + row] : p.stack[have - 1 - (s_need[b] + row - held)];
        if (page >= 0) slot = (int64_t)page * p.page + (pos - row * p.page);
      }
    }
    p.slots[t] = slot;
    p.positions[t] = pos;
  }
}

__global__ __launch_bounds__(256) void bt_tokens(Params p, int per_block) {
  extern __shared__ int s_cu[];
  for (int b = threadIdx.x; b <= p.batch; b += 256) s_cu[b] = p.cu[b];
  __syncthreads();
  const int64_t first = (int64_t)blockIdx.x * per_block;
  const int64_t end = min(first + per_block, (int64_t)p.tokens);
  for (int64_t t = first + threadIdx.x; t < end; t += 256) {
    int64_t slot = -1, pos = 0;
    if (t < s_cu[p.batch]) {
      const int b = find(s_cu, p.batch, (int)t);
      const int cached = max(p.cached[b], 0);
      pos = (int64_t)cached + (t - s_cu[b]);
      const int64_t row = div_page(p, (uint32_t)pos);
      // (a request with tokens is served if and only if its length has grown; its pages are in the table)
      const int page = p.seq_lens[b] != cached ? p.table[b * p.t_sr + row] : -1;
      if (page >= 0) slot = (int64_t)page * p.page + (pos - row * p.page);
    }
    p.slots[t] = slot;
    p.positions[t] = pos;
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
  if (a->batch > 1 && a->bt_stride_row < a->table_pages)
    return set_error(L20_PD_EINVAL, "block table rows overlap");
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
  p.magic = l20bt::page_magic((uint32_t)p.page);
  p.inline_tokens = a->num_slots <= l20bt::kTokensInline;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const size_t lds = (size_t)(4 * (a->batch + 1)) * sizeof(int);  // at most 128 KB
  static l20la::LdsLimit limit;
  const int most = 4 * (L20_PD_MAX_REQUESTS + 1) * (int)sizeof(int);
  const hipError_t e = limit.raise(reinterpret_cast<const void *>(&l20bt::bt_requests), most);
  if (e != hipSuccess) return set_error(L20_PD_ELAUNCH, hipGetErrorString(e));
  hipLaunchKernelGGL(l20bt::bt_requests, dim3(1), dim3(l20bt::kThreads), lds, s, p);
  int32_t r = launched();
  if (r != L20_PD_OK || p.inline_tokens) return r;
  const int per_block = 256;
  hipLaunchKernelGGL(l20bt::bt_tokens, dim3((unsigned)(((int64_t)p.tokens + per_block - 1) / per_block)), dim3(256),
                     (size_t)(a->batch + 1) * sizeof(int), s, p, per_block);
  return launched();
}

}  // extern "C"
