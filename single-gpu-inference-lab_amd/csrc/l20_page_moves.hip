// The page pool of a paged cache (gfx950): rows of the block table that follow their parents, the pool's
// compaction, and the copies of pages that both ask for.
//
//  rp_cells   a wave a group of beams and 64 columns of its rows, a lane a column.  All of a column's cells are in
//    LDS before any is written, so rows exchange in place.  What the group's holders of a page change is added to
//    page_shares in one atomic: the sum reaches -1 in the one atomic after which no row anywhere holds the page (a
//    group only adds holders to pages that it holds), whatever the order.  Freed pages go to a list a wave.
//  rp_pool    one workgroup.  The freed pages are put into a bitmap, so that they go on the stack by number and not
//    by the order of atomics; then the rows that need a copy take theirs, by two scans.
//  cp_clear, cp_mark, cp_scan, cp_remap   pages to move and pages to move to as bitmaps, their ranks by one
//    workgroup's scan, and the table's cells after them.
//  pc_copy    workgroups take (pair, cache, 16 KB) in turn.

#include "l20_block_tables.h"

#include <algorithm>

#include "l20_beam_search.h"
#include "l20_latent_common.h"

namespace l20pm {

using l20la::i32x2;
using l20la::i32x4;

constexpr int kThreads = 1024;
constexpr int kPerThread = L20_PD_MAX_REQUESTS / kThreads;
constexpr int kCellWaves = 4;
constexpr int kBitmap = 1 << 19;  // pages of one pass of rp_pool (64 KB of LDS)
constexpr int kUnits = 8192;      // waves' lists that rp_pool looks at together

__device__ __forceinline__ int pages_of(int tokens, int page) { return tokens > 0 ? (int)(((int64_t)tokens + page - 1) / page) : 0; }

// Inclusive scan of a value a thread over the workgroup; `total` is the sum.
__device__ __forceinline__ int scan(int x, int *s_wave, int &total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const int y = __shfl_up(x, off);
    if (lane >= off) x += y;
  }
  __syncthreads();
  if (lane == 63) s_wave[wave] = x;
  __syncthreads();
  total = 0;
#pragma unroll
  for (int w = 0; w < kThreads / 64; ++w) {
    const int v = s_wave[w];
    x += w < wave ? v : 0;
    total += v;
  }
  return x;
}

struct Reorder {
  const int32_t *parents;
  int32_t *table;
  int64_t t_sr;
  int width;
  int32_t *lens;
  int32_t *shares;
  int pages;
  int32_t *stack;
  int pool;
  int32_t *count;
  int32_t *src, *dst, *tokens;
  int room;
  int32_t *pairs;
  int groups, beams, page;
  int blocks;           // of 64 columns
  int32_t *list_count;  // [groups * blocks]
  int32_t *list;        // [groups * blocks][beams * 64]
  int32_t *source;      // [groups * beams] the page that a row's copy comes from
};

// What becomes of a row, from its group's parents and lengths (a lane a row).
struct Row {
  int parent;  // -1: given up
  int len;     // new
  int copy;    // the column of its own copy, -1: none
};
__device__ __forceinline__ Row row_of(int row, int beams, int parent, int parent_len, bool parent_stays, bool first, int page, int width) {
  Row r{parent, parent >= 0 ? max(parent_len, 0) : 0, -1};
  const bool keeps = parent_stays ? parent == row : first;
  if (parent >= 0 && r.len % page != 0 && !keeps && r.len / page < width) r.copy = r.len / page;
  return r;
}

__global__ __launch_bounds__(64 * kCellWaves) void rp_cells(Reorder p) {
  extern __shared__ int s_cells[];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int group = blockIdx.y, block = blockIdx.x * kCellWaves + wave;
  if (block >= p.blocks) return;
  const int beams = p.beams, c = block * 64 + lane;
  int *const mine = s_cells + wave * beams * 64 + lane;  // this lane's column: [beams], 64 apart
  // a lane a row
  const int known = min(lane, beams - 1), at = group * beams + known;
  const int old_len = max(p.lens[at], 0);
  int parent = p.parents[at];
  if (parent < 0 || parent >= beams) parent = -1;
  const int from = max(parent, 0);
  const int parent_len = __shfl(old_len, from), grandparent = __shfl(parent, from);  // (by every lane)
  const bool stays = parent >= 0 && grandparent == parent;
  bool first = true;
  for (int i = 0; i < beams; ++i) {
    const int other = __builtin_amdgcn_readlane(parent, i);
    if (i < lane && other == parent) first = false;
  }
  const Row row = row_of(known, beams, parent, parent_len, stays, first, p.page, p.width);
  const int held = min(pages_of(old_len, p.page), p.width), new_held = min(pages_of(row.len, p.page), p.width);
  int32_t *const cells = p.table + (int64_t)group * beams * p.t_sr + c;
  auto has = [&](int i) { return c < __builtin_amdgcn_readlane(held, i); };
  for (int i = 0; i < beams; ++i) mine[i * 64] = has(i) ? cells[i * p.t_sr] : -1;
  // whether row i takes its parent's cell (not its own copy's, and none beyond its length), and what that is, else -1
  auto next = [&](int i, int &v) {
    const int q = __builtin_amdgcn_readlane(row.parent, i);
    const bool follows = q >= 0 && c < __builtin_amdgcn_readlane(new_held, i) && c != __builtin_amdgcn_readlane(row.copy, i);
    v = follows ? mine[q * 64] : -1;
    return follows;
  };
  bool any = false;
  for (int i = 0; i < beams; ++i) {
    const int q = __builtin_amdgcn_readlane(row.parent, i), copy = __builtin_amdgcn_readlane(row.copy, i);
    if (q >= 0 && c == copy) p.source[group * beams + i] = mine[q * 64];
    int v;
    any |= next(i, v) != has(i) || v != mine[i * 64];
  }
  const int unit = group * p.blocks + block;
  int listed = 0;
  if (__ballot(any)) {
    int32_t *const list = p.list + (int64_t)unit * beams * 64;
    for (int r = 0; r < beams; ++r) {
      const int v = mine[r * 64];
      bool gone = false;
      if (any && v >= 0 && v < p.pages) {
        int change = 0;
        bool seen = false;  // in an earlier row: counted there
        for (int i = 0; i < beams; ++i) {
          const bool same = mine[i * 64] == v;
          int w;
          next(i, w);
          seen |= same && i < r;
          change += (w == v) - same;
        }
        if (!seen && change != 0) gone = atomicAdd(p.shares + v, change) + change == -1;
        if (gone) p.shares[v] = 0;
      }
      const unsigned long long which = __ballot(gone);
      if (gone) list[listed + __builtin_popcountll(which & (((unsigned long long)1 << lane) - 1))] = v;
      listed += __builtin_popcountll(which);
    }
    for (int i = 0; i < beams; ++i) {
      int v;
      if (next(i, v) && (!has(i) || v != mine[i * 64])) cells[i * p.t_sr] = v;
    }
  }
  if (lane == 0) p.list_count[unit] = listed;
}

__global__ __launch_bounds__(kThreads) void rp_pool(Reorder p) {
  extern __shared__ int s_mem[];
  __shared__ int s_wave[kThreads / 64];
  unsigned int *const s_bits = (unsigned int *)s_mem;  // [min(pages, kBitmap) / 32]
  int *const s_at = s_mem + (min(p.pages, kBitmap) + 31) / 32;  // [kUnits + 1]: list offsets, then the parents
  int *const s_len = s_at + kUnits + 1;                         // [rows] old lengths
  const int tid = threadIdx.x, rows = p.groups * p.beams, units = p.groups * p.blocks;
  const int count = min(max(*p.count, 0), p.pool);
  for (int r = tid; r < rows; r += kThreads) s_len[r] = p.lens[r];
  // freed pages onto the stack, by number
  int freed = 0;
  for (int base = 0; base < p.pages; base += kBitmap) {
    const int n = min(p.pages - base, kBitmap), words = (n + 31) / 32;
    for (int i = tid; i < words; i += kThreads) s_bits[i] = 0;
    bool some = false;
    for (int u0 = 0; u0 < units; u0 += kUnits) {
      const int here = min(units - u0, kUnits), per = (here + kThreads - 1) / kThreads;
      int mine = 0;
      for (int i = 0; i < per; ++i) {
        const int u = tid * per + i;
        if (u < here) mine += p.list_count[u0 + u];
      }
      int total;
      int at = scan(mine, s_wave, total) - mine;  // (its barriers: the bitmap is clear, the offsets are read)
      if (total == 0) continue;
      some = true;
      for (int i = 0; i < per; ++i) {
        const int u = tid * per + i;
        if (u < here) {
          s_at[u] = at;
          at += p.list_count[u0 + u];
        }
      }
      if (tid == 0) s_at[here] = total;
      __syncthreads();
      for (int k = tid; k < total; k += kThreads) {
        int lo = 0, hi = here - 1;
        while (lo < hi) {
          const int mid = (lo + hi + 1) >> 1;
          if (s_at[mid] <= k) lo = mid;
          else hi = mid - 1;
        }
        const int v = p.list[(int64_t)(u0 + lo) * p.beams * 64 + (k - s_at[lo])] - base;
        if (v >= 0 && v < n) atomicOr(s_bits + (v >> 5), 1u << (v & 31));
      }
    }
    __syncthreads();
    if (!some) break;  // (the same lists for every base)
    const int per = (words + kThreads - 1) / kThreads;
    int mine = 0;
    for (int i = 0; i < per; ++i)
      if (tid * per + i < words) mine += __builtin_popcount(s_bits[tid * per + i]);
    int total;
    int64_t at = (int64_t)count + freed + scan(mine, s_wave, total) - mine;
    for (int i = 0; i < per && tid * per + i < words; ++i)
      for (unsigned int w = s_bits[tid * per + i]; w; w &= w - 1, ++at)
        if (at < p.pool) p.stack[at] = base + (tid * per + i) * 32 + __builtin_ctz(w);
    freed += total;
    __syncthreads();
  }
  const int have = (int)min((int64_t)count + freed, (int64_t)p.pool);
  __syncthreads();
  // rows that need a page, in order
  int *const s_parent = s_at;
  for (int r = tid; r < rows; r += kThreads) s_parent[r] = p.parents[r];
  __syncthreads();
  const int per = (rows + kThreads - 1) / kThreads;
  Row row[kPerThread];
  int wanted = 0;
#pragma unroll
  for (int i = 0; i < kPerThread; ++i) {
    const int r = tid * per + i;
    row[i] = Row{-1, 0, -1};
    if (i < per && r < rows) {
      const int group = r / p.beams, me = r - group * p.beams;
      const int *const family = s_parent + group * p.beams;
      int parent = family[me];
      if (parent < 0 || parent >= p.beams) parent = -1;
      bool first = true;
      for (int j = 0; j < me; ++j) first &= family[j] != parent;
      row[i] = row_of(me, p.beams, parent, s_len[group * p.beams + max(parent, 0)], parent >= 0 && family[parent] == parent, first,
                      p.page, p.width);
      wanted += row[i].copy >= 0;
    }
  }
  int total;
  int64_t k = scan(wanted, s_wave, total) - wanted;
  int got[kPerThread], served = 0;
#pragma unroll
  for (int i = 0; i < kPerThread; ++i) {
    const int r = tid * per + i;
    got[i] = -1;
    if (i < per && r < rows) {
      p.lens[r] = row[i].len;
      if (row[i].copy >= 0) {
        if (k < have) got[i] = p.stack[have - 1 - k];
        ++k;
        if (got[i] < 0 || got[i] >= p.pages) got[i] = -1;
        p.table[r * p.t_sr + row[i].copy] = got[i];
        served += got[i] >= 0;
      }
    }
  }
  int pairs;
  int at = scan(served, s_wave, pairs) - served;
#pragma unroll
  for (int i = 0; i < kPerThread; ++i) {
    const int r = tid * per + i;
    if (i < per && r < rows && got[i] >= 0) {
      p.src[at] = p.source[r];
      p.dst[at] = got[i];
      p.tokens[at] = row[i].len % p.page;
      ++at;
    }
  }
  for (int i = pairs + tid; i < p.room; i += kThreads) p.src[i] = -1, p.dst[i] = -1, p.tokens[i] = 0;
  if (tid == 0) {
    p.pairs[0] = pairs;
    p.pairs[1] = total - pairs;
    *p.count = have - min(total, have);
  }
}

struct Compact {
  int limit;
  int32_t *table;
  int64_t t_sr;
  int width;
  const int32_t *lens;
  int32_t *shares;
  int pages;
  int32_t *stack;
  int pool;
  int32_t *count;
  int32_t *src, *dst, *tokens;
  int room;
  int32_t *pairs;
  int rows, page;
  int words;            // of a bitmap of the pages
  unsigned int *high;   // pages held at or beyond the limit
  unsigned int *low;    // free ones below it
  int32_t *map;         // [pages] where a page of `high` goes
  int row_blocks;       // of 256 columns, a row
};

__global__ __launch_bounds__(256) void cp_clear(Compact p) {
  const int i = blockIdx.x * 256 + threadIdx.x;
  if (i < p.words) p.high[i] = p.low[i] = 0;
}

__global__ __launch_bounds__(256) void cp_mark(Compact p) {
  const int64_t tables = (int64_t)p.rows * p.row_blocks;
  if (blockIdx.x < tables) {
    const int row = (int)(blockIdx.x / p.row_blocks), c = (int)(blockIdx.x % p.row_blocks) * 256 + threadIdx.x;
    if (c >= min(pages_of(p.lens[row], p.page), p.width)) return;
    const int v = p.table[row * p.t_sr + c];
    if (v >= p.limit && v < p.pages) atomicOr(p.high + (v >> 5), 1u << (v & 31));
  } else {
    const int64_t i = (blockIdx.x - tables) * 256 + threadIdx.x;
    if (i >= min(max(*p.count, 0), p.pool)) return;
    const int v = p.stack[i];
    if (v >= 0 && v < p.limit) atomicOr(p.low + (v >> 5), 1u << (v & 31));
  }
}

__global__ __launch_bounds__(kThreads) void cp_scan(Compact p) {
  __shared__ int s_wave[kThreads / 64];
  const int tid = threadIdx.x, per = (p.words + kThreads - 1) / kThreads;
  int highs = 0, lows = 0;
  for (int i = 0; i < per; ++i)
    if (tid * per + i < p.words) {
      highs += __builtin_popcount(p.high[tid * per + i]);
      lows += __builtin_popcount(p.low[tid * per + i]);
    }
  int all_high, all_low;
  int high = scan(highs, s_wave, all_high) - highs, low = scan(lows, s_wave, all_low) - lows;
  const int moves = min(min(all_high, all_low), p.room);
  for (int i = 0; i < per && tid * per + i < p.words; ++i) {
    const int base = (tid * per + i) * 32;
    for (unsigned int w = p.high[tid * per + i]; w; w &= w - 1, ++high) {
      const int v = base + __builtin_ctz(w);
      if (high < moves) p.src[high] = v;
      else p.map[v] = v;
    }
    for (unsigned int w = p.low[tid * per + i]; w; w &= w - 1, ++low) {
      const int v = base + __builtin_ctz(w);
      if (low < moves) p.dst[low] = v;
      else if (all_low - 1 - low < p.pool) p.stack[all_low - 1 - low] = v;
    }
  }
  __syncthreads();
  for (int k = tid; k < p.room; k += kThreads) {
    if (k < moves) {
      const int from = p.src[k], to = p.dst[k];
      p.map[from] = to;
      p.shares[to] = p.shares[from];
      p.shares[from] = 0;
      p.tokens[k] = p.page;
    } else {
      p.src[k] = -1, p.dst[k] = -1, p.tokens[k] = 0;
    }
  }
  if (tid == 0) {
    *p.count = all_low - moves;
    p.pairs[0] = moves;
    p.pairs[1] = all_high - moves;
  }
}

__global__ __launch_bounds__(256) void cp_remap(Compact p) {
  const int row = (int)(blockIdx.x / p.row_blocks), c = (int)(blockIdx.x % p.row_blocks) * 256 + threadIdx.x;
  if (c >= min(pages_of(p.lens[row], p.page), p.width)) return;
  int32_t *const cell = p.table + row * p.t_sr + c;
  const int v = *cell;
  if (v >= p.limit && v < p.pages) *cell = p.map[v];
}

constexpr int kCaches = 64;  // caches of a launch

struct Copy {
  const int32_t *src, *dst, *tokens;
  int room;
  const int32_t *count;
  char *cache[kCaches];
  int caches;
  int64_t pages, page_stride;
  int64_t size[3], stride[3], inner;  // levels outside in; inner: contiguous bytes
  int token_level;
  int64_t units;    // of one page, each sizeof(V) bytes
  int64_t segment;  // units a workgroup takes at once
  int segments;     // of a page
};

// DENSE: a page is one run of bytes, and its first tokens the first bytes.
template <typename V, bool DENSE> __global__ __launch_bounds__(256) void pc_copy(Copy p) {
  const int pairs = p.count ? min(max(*p.count, 0), p.room) : p.room;
  const int64_t all = (int64_t)pairs * p.caches * p.segments;
  const int64_t inner = p.inner / (int64_t)sizeof(V);
  for (int64_t job = blockIdx.x; job < all; job += gridDim.x) {
    const int segment = (int)(job % p.segments);
    const int64_t rest = job / p.segments;
    const int cache = (int)(rest % p.caches), pair = (int)(rest / p.caches);
    const int from = p.src[pair], to = p.dst[pair];
    if (from < 0 || from >= p.pages || to < 0 || to >= p.pages) continue;
    int64_t tokens = INT64_MAX;
    if (p.token_level >= 0 && p.tokens) tokens = max(p.tokens[pair], 0);
    const char *const a = p.cache[cache] + from * p.page_stride;
    char *const b = p.cache[cache] + to * p.page_stride;
    int64_t end = min(((int64_t)segment + 1) * p.segment, p.units);
    if constexpr (DENSE) {
      if (p.token_level >= 0) end = min(end, min(tokens, p.size[0]) * (p.stride[0] / (int64_t)sizeof(V)));
      for (int64_t i = segment * p.segment + threadIdx.x; i < end; i += 4 * 256) {
        V v[4];
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (i + j * 256 < end) v[j] = reinterpret_cast<const V *>(a)[i + j * 256];
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (i + j * 256 < end) reinterpret_cast<V *>(b)[i + j * 256] = v[j];
      }
    } else {
      for (int64_t i = segment * p.segment + threadIdx.x; i < end; i += 256) {
        const int64_t x = i / inner, x2 = x % p.size[2], y = x / p.size[2], x1 = y % p.size[1], x0 = y / p.size[1];
        const int64_t token = p.token_level == 0 ? x0 : p.token_level == 1 ? x1 : p.token_level == 2 ? x2 : 0;
        if (token >= tokens) continue;
        const int64_t at = x0 * p.stride[0] + x1 * p.stride[1] + x2 * p.stride[2] + (i - x * inner) * (int64_t)sizeof(V);
        *reinterpret_cast<V *>(b + at) = *reinterpret_cast<const V *>(a + at);
      }
    }
  }
}

}  // namespace l20pm

namespace {

using l20pd_host::set_error;

bool bad_page(int32_t page) { return page < 16 || page % 16 || page > 4096; }
constexpr const char *kBadPage = "page size must be a multiple of 16 up to 4096";
constexpr int64_t kMaxCells = (int64_t)1 << 30;

int32_t check(const l20_pd_reorder_args *a) {
  if (!a) return set_error(L20_PD_EINVAL, "null argument block");
  if (a->beams < 1 || a->beams > L20_PD_MAX_BEAMS) return set_error(L20_PD_EINVAL, "1 to 32 beams");
  if (a->groups < 0 || (int64_t)a->groups * a->beams > L20_PD_MAX_REQUESTS)
    return set_error(L20_PD_EINVAL, "block tables: at most 8192 rows");
  if (bad_page(a->page_size)) return set_error(L20_PD_EINVAL, kBadPage);
  if (a->pages < 1 || a->pool < 1 || (a->groups > 0 && a->table_pages < 1))
    return set_error(L20_PD_EINVAL, "block table and page pool must not be empty");
  const int64_t rows = (int64_t)a->groups * a->beams;
  if (a->pages > kMaxCells || a->pool > kMaxCells || rows * (((int64_t)a->table_pages + 63) / 64 * 64) > kMaxCells)
    return set_error(L20_PD_EINVAL, "block table or page pool too large");
  if (a->room < rows) return set_error(L20_PD_EINVAL, "room for a pair a row is needed");
  if (!a->page_shares || !a->free_pages || !a->free_count || !a->count ||
      (rows > 0 && (!a->parents || !a->block_table || !a->seq_lens || !a->src || !a->dst || !a->tokens)))
    return set_error(L20_PD_EINVAL, "null tensor pointer");
  if (rows > 1 && a->bt_stride_row < a->table_pages) return set_error(L20_PD_EINVAL, "block table rows overlap");
  return L20_PD_OK;
}

int64_t workspace(const l20_pd_reorder_args *a) {
  const int64_t blocks = ((int64_t)a->table_pages + 63) / 64;
  return 4 * (a->groups * blocks * (1 + (int64_t)a->beams * 64) + (int64_t)a->groups * a->beams);
}

int32_t check(const l20_pd_compact_args *a) {
  if (!a) return set_error(L20_PD_EINVAL, "null argument block");
  if (a->rows < 0 || a->rows > L20_PD_MAX_REQUESTS) return set_error(L20_PD_EINVAL, "block tables: at most 8192 rows");
  if (bad_page(a->page_size)) return set_error(L20_PD_EINVAL, kBadPage);
  if (a->pages < 1 || a->pool < 1 || (a->rows > 0 && a->table_pages < 1))
    return set_error(L20_PD_EINVAL, "block table and page pool must not be empty");
  if (a->pages > kMaxCells || a->pool > kMaxCells || (int64_t)a->rows * a->table_pages > kMaxCells)
    return set_error(L20_PD_EINVAL, "block table or page pool too large");
  if (a->limit < 0 || a->limit > a->pages) return set_error(L20_PD_EINVAL, "limit must be 0 to the number of pages");
  if (a->room < 0) return set_error(L20_PD_EINVAL, "room must not be negative");
  if (!a->page_shares || !a->free_pages || !a->free_count || !a->count || (a->rows > 0 && (!a->block_table || !a->seq_lens)) ||
      (a->room > 0 && (!a->src || !a->dst || !a->tokens)))
    return set_error(L20_PD_EINVAL, "null tensor pointer");
  if (a->rows > 1 && a->bt_stride_row < a->table_pages) return set_error(L20_PD_EINVAL, "block table rows overlap");
  return L20_PD_OK;
}

int64_t words_of(const l20_pd_compact_args *a) { return ((int64_t)a->pages + 31) / 32; }

int32_t check(const l20_pd_copy_args *a) {
  if (!a) return set_error(L20_PD_EINVAL, "null argument block");
  if (a->room < 0 || a->num_caches < 0) return set_error(L20_PD_EINVAL, "pairs and caches must not be negative");
  if (a->pages < 1 || a->size0 < 1 || a->size1 < 1 || a->size2 < 1 || a->inner < 1)
    return set_error(L20_PD_EINVAL, "cache must not be empty");
  if (a->token_level < -1 || a->token_level > 2) return set_error(L20_PD_EINVAL, "token level must be -1 to 2");
  const int64_t size[3] = {a->size0, a->size1, a->size2}, stride[3] = {a->stride0, a->stride1, a->stride2};
  int64_t below = a->inner;  // bytes that a step of the level inside spans: levels must not run into each other
  for (int i = 2; i >= 0; --i) {
    if (size[i] > kMaxCells || below > ((int64_t)1 << 40)) return set_error(L20_PD_EINVAL, "page too large");
    if (size[i] > 1) {
      if (stride[i] < below || stride[i] > ((int64_t)1 << 40)) return set_error(L20_PD_EINVAL, "a page's parts overlap");
      below = (size[i] - 1) * stride[i] + below;
    }
  }
  if (a->pages > 1 && a->stride_page < 1) return set_error(L20_PD_EINVAL, "pages overlap");
  if (a->room == 0 || a->num_caches == 0) return L20_PD_OK;
  if (!a->src || !a->dst || !a->caches) return set_error(L20_PD_EINVAL, "null tensor pointer");
  for (int i = 0; i < a->num_caches; ++i)
    if (!a->caches[i]) return set_error(L20_PD_EINVAL, "null tensor pointer");
  return L20_PD_OK;
}

int32_t launched() {
  const hipError_t e = hipGetLastError();
  if (e == hipSuccess) return L20_PD_OK;
  char msg[256];
  snprintf(msg, sizeof(msg), "HIP launch failed: %s", hipGetErrorString(e));
  return set_error(L20_PD_ELAUNCH, msg);
}

template <typename V> int32_t launch_copy(const l20pm::Copy &p, bool dense, hipStream_t s) {
  const int64_t jobs = (int64_t)p.room * p.caches * p.segments;
  const unsigned grid = (unsigned)std::min<int64_t>(jobs, 8 * (int64_t)l20la::device_cus());
  if (dense) hipLaunchKernelGGL((l20pm::pc_copy<V, true>), dim3(grid), dim3(256), 0, s, p);
  else hipLaunchKernelGGL((l20pm::pc_copy<V, false>), dim3(grid), dim3(256), 0, s, p);
  return launched();
}

}  // namespace

extern "C" {

int32_t l20_pd_reorder_tables_check(const l20_pd_reorder_args *a) {
  l20pd_host::clear_error();
  return check(a);
}

int64_t l20_pd_reorder_tables_workspace(const l20_pd_reorder_args *a) {
  return a && a->groups > 0 && a->beams > 0 && a->table_pages > 0 ? workspace(a) : 0;
}

int32_t l20_pd_reorder_tables(const l20_pd_reorder_args *a, void *stream) {
  l20pd_host::clear_error();
  int32_t rc = check(a);
  if (rc != L20_PD_OK) return rc;
  if (a->groups > 0 && (!a->workspace || (uintptr_t)a->workspace % 4 || a->workspace_bytes < workspace(a)))
    return set_error(L20_PD_EINVAL, "workspace is missing, misaligned or too small");
  l20pm::Reorder p{};
  p.parents = a->parents;
  p.table = a->block_table;
  p.t_sr = a->bt_stride_row;
  p.width = a->table_pages;
  p.lens = a->seq_lens;
  p.shares = a->page_shares;
  p.pages = a->pages;
  p.stack = a->free_pages;
  p.pool = a->pool;
  p.count = a->free_count;
  p.src = a->src;
  p.dst = a->dst;
  p.tokens = a->tokens;
  p.room = a->room;
  p.pairs = a->count;
  p.groups = a->groups;
  p.beams = a->beams;
  p.page = a->page_size;
  p.blocks = (a->table_pages + 63) / 64;
  p.list_count = reinterpret_cast<int32_t *>(a->workspace);
  p.list = p.list_count + (int64_t)p.groups * p.blocks;
  p.source = p.list + (int64_t)p.groups * p.blocks * p.beams * 64;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  if (p.groups > 0) {
    const dim3 grid((unsigned)((p.blocks + l20pm::kCellWaves - 1) / l20pm::kCellWaves), (unsigned)p.groups);
    hipLaunchKernelGGL(l20pm::rp_cells, grid, dim3(64 * l20pm::kCellWaves), (size_t)l20pm::kCellWaves * p.beams * 256, s, p);
    rc = launched();
    if (rc != L20_PD_OK) return rc;
  }
  const auto pool_lds = [](int64_t pages, int64_t rows) {
    return (int)(4 * ((std::min<int64_t>(pages, l20pm::kBitmap) + 31) / 32 + l20pm::kUnits + 1 + rows));
  };
  static l20la::LdsLimit limit;
  const hipError_t e = limit.raise(reinterpret_cast<const void *>(&l20pm::rp_pool), pool_lds(l20pm::kBitmap, L20_PD_MAX_REQUESTS));
  if (e != hipSuccess) return set_error(L20_PD_ELAUNCH, hipGetErrorString(e));
  hipLaunchKernelGGL(l20pm::rp_pool, dim3(1), dim3(l20pm::kThreads), (size_t)pool_lds(p.pages, (int64_t)p.groups * p.beams), s, p);
  return launched();
}

int32_t l20_pd_compact_pages_check(const l20_pd_compact_args *a) {
  l20pd_host::clear_error();
  return check(a);
}

int64_t l20_pd_compact_pages_workspace(const l20_pd_compact_args *a) {
  return a && a->pages > 0 ? 4 * (2 * words_of(a) + a->pages) : 0;
}

int32_t l20_pd_compact_pages(const l20_pd_compact_args *a, void *stream) {
  l20pd_host::clear_error();
  int32_t rc = check(a);
  if (rc != L20_PD_OK) return rc;
  if (!a->workspace || (uintptr_t)a->workspace % 4 || a->workspace_bytes < l20_pd_compact_pages_workspace(a))
    return set_error(L20_PD_EINVAL, "workspace is missing, misaligned or too small");
  l20pm::Compact p{};
  p.limit = a->limit;
  p.table = a->block_table;
  p.t_sr = a->bt_stride_row;
  p.width = a->table_pages;
  p.lens = a->seq_lens;
  p.shares = a->page_shares;
  p.pages = a->pages;
  p.stack = a->free_pages;
  p.pool = a->pool;
  p.count = a->free_count;
  p.src = a->src;
  p.dst = a->dst;
  p.tokens = a->tokens;
  p.room = a->room;
  p.pairs = a->count;
  p.rows = a->rows;
  p.page = a->page_size;
  p.words = (int)words_of(a);
  p.high = reinterpret_cast<unsigned int *>(a->workspace);
  p.low = p.high + p.words;
  p.map = reinterpret_cast<int32_t *>(p.low + p.words);
  p.row_blocks = std::max(1, (a->table_pages + 255) / 256);
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const int64_t tables = (int64_t)p.rows * p.row_blocks, stacks = ((int64_t)p.pool + 255) / 256;
  hipLaunchKernelGGL(l20pm::cp_clear, dim3((unsigned)((p.words + 255) / 256)), dim3(256), 0, s, p);
  hipLaunchKernelGGL(l20pm::cp_mark, dim3((unsigned)(tables + stacks)), dim3(256), 0, s, p);
  hipLaunchKernelGGL(l20pm::cp_scan, dim3(1), dim3(l20pm::kThreads), 0, s, p);
  if (tables > 0) hipLaunchKernelGGL(l20pm::cp_remap, dim3((unsigned)tables), dim3(256), 0, s, p);
  return launched();
}

int32_t l20_pd_copy_pages_check(const l20_pd_copy_args *a) {
  l20pd_host::clear_error();
  return check(a);
}

int32_t l20_pd_copy_pages(const l20_pd_copy_args *a, void *stream) {
  l20pd_host::clear_error();
  int32_t rc = check(a);
  if (rc != L20_PD_OK || a->room == 0 || a->num_caches == 0) return rc;
  l20pm::Copy p{};
  p.src = a->src;
  p.dst = a->dst;
  p.tokens = a->tokens;
  p.room = a->room;
  p.count = a->count;
  p.pages = a->pages;
  p.page_stride = a->pages > 1 ? a->stride_page : 0;
  p.inner = a->inner;
  p.token_level = a->tokens ? a->token_level : -1;
  const int64_t size[3] = {a->size0, a->size1, a->size2}, stride[3] = {a->stride0, a->stride1, a->stride2};
  // widest units that every address is a multiple of
  uint64_t low = (uint64_t)p.inner | (uint64_t)p.page_stride;
  int64_t bytes = p.inner;
  bool dense = true;
  for (int i = 2; i >= 0; --i) {
    p.size[i] = size[i];
    p.stride[i] = size[i] > 1 ? stride[i] : bytes;  // (of one step: as if dense)
    dense &= p.stride[i] == bytes;
    if (size[i] > 1) low |= (uint64_t)stride[i];
    bytes *= size[i];
  }
  dense &= p.token_level <= 0;
  for (int i = 0; i < a->num_caches; ++i) low |= (uint64_t)(uintptr_t)a->caches[i];
  const int unit = low % 16 == 0 ? 16 : low % 8 == 0 ? 8 : low % 4 == 0 ? 4 : low % 2 == 0 ? 2 : 1;
  p.units = bytes / unit;
  p.segment = std::min<int64_t>(p.units, 1024);
  p.segments = (int)((p.units + p.segment - 1) / p.segment);
  for (int first = 0; first < a->num_caches && rc == L20_PD_OK; first += l20pm::kCaches) {
    p.caches = std::min(l20pm::kCaches, a->num_caches - first);
    for (int i = 0; i < p.caches; ++i) p.cache[i] = reinterpret_cast<char *>(a->caches[first + i]);
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    rc = unit == 16  ? launch_copy<l20la::i32x4>(p, dense, s)
         : unit == 8 ? launch_copy<l20la::i32x2>(p, dense, s)
         : unit == 4 ? launch_copy<int32_t>(p, dense, s)
         : unit == 2 ? launch_copy<int16_t>(p, dense, s)
                     : launch_copy<int8_t>(p, dense, s);
  }
  return rc;
}

}  // extern "C"
