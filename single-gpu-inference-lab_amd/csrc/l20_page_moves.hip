// The page pool of a paged cache (gfx950): rows of the block table that follow their parents, the pool's
// compaction, and the copies of pages that both ask for.
//
//  rp_cells   a wave a group of beams and 64 columns of its rows, a lane a column.  All of a column's cells are in
//    LDS before any is written, so rows exchange in place; the changes of page_shares are atomics whose order does
//    not matter.  Freed pages go to a list a wave.
//  rp_pool    one workgroup.  Freed pages go on the stack by number, not by the order of atomics, through a bitmap in
//    LDS; then the rows that need a copy take theirs.
//  rp_small   both in one launch.
//  cp_clear, cp_mark, cp_place, cp_remap   pages to move and pages to move to as bitmaps; a page's rank among them,
//    and so its place, from the bits before it; the table's cells by the ranks.  cp_small: all of it in one launch.
//  pc_copy    workgroups take (pair, cache, 16 KB) in turn.
//
// What bounds them: for all but the copies the latency of a few dependent loads, not bytes (kernel times).
//  rp_cells   64 groups of 4 beams of 4000-8000 tokens (0.4 MB of cells) 5.8 us: lengths and parents, cells, atomics of
//    page_shares in two waves (gains, losses), cells.  24 groups of 16 beams, a quarter given back, 8.9: up to 16 atomics
//    a lane, eight in flight (two, four, 16 at once: 1.7 and 0.6 us more, and 4.5: small calls and single waves wait for code
//    as much as for data, and 16 are too much of it).
//  rp_pool    5.3-7.2 us: lists' lengths, their entries, two scans, the stack; one workgroup, since its answer is an order.
//  rp_small   4 groups of 4 beams 6.9 us, both chains one behind the other.
//  cp_clear, cp_mark, cp_place, cp_remap   256 rows, a pool of 200000 pages 2.0 + 6.8 + 6.6 + 3.3 us: launches, 200000 atomics
//    on the bitmaps, and counting before placing.  cp_small: 16 rows, 4096 pages 5.7 us.
//  pc_copy    memory: 512 whole pages of 16 tokens of 56 caches (470 MB read and written) 198 us, 4.75 TB/s (a library copy of
//    1 GiB 5.12); 12 pages in part of 56 fp8 caches 4.3 us.

#include "l20_block_tables.h"

#include <algorithm>

#include "l20_beam_search.h"
#include "l20_latent_common.h"
#include "l20_overlap.h"

namespace l20pm {

using l20la::i32x2;
using l20la::i32x4;
using l20la::wave_scan;

constexpr int kThreads = 1024;
constexpr int kPerThread = L20_PD_MAX_REQUESTS / kThreads;
constexpr int kCellWaves = 4;
constexpr int kBitmap = 1 << 18;  // pages of one pass of rp_pool (32 KB of LDS)
constexpr int kUnits = 4096;      // waves' lists that rp_pool looks at together
// Waves' worth of cells that one launch does with the pool, one a wave.  Measured against two launches: 8 groups of 4
// beams, 64 cells 9.8 and 13.1 us, 16 groups 11.8 and 13.7; more than one a wave, 32 groups 17.3 and 13.0.
constexpr int kSmall = 16;
// Pages, and waves' worth of cells, of a compaction in one launch.  Measured against four: 64 rows of 64 cells, 8192 pages
// 13.1 and 17.4 us, 16 of 128, 4096 pages 8.2 and 16.8; beyond, 64 rows of 256, 20000 pages 28.1 and 17.4, 256 rows of 64,
// 30000 pages 40.6 and 17.7.
constexpr int kSmallPages = 1 << 13, kSmallWaves = 64;

// A page of 16 d tokens, and division by it: of n / 16 below 2^28 by d as a product with ceil(2^(28 + l) / d), 2^l >= d, whose
// excess is below 2^-l.  (The compiler's divisions are long, and code is what small calls wait for.)
struct Page {
  int size;
  uint32_t mul;
  int shift;
  Page(int size_ = 16) : size(size_), shift(28) {
    const uint64_t d = (uint64_t)size / 16;
    while (((uint64_t)1 << (shift - 28)) < d) ++shift;
    mul = (uint32_t)((((uint64_t)1 << shift) + d - 1) / d);
  }
  __device__ __forceinline__ int whole(unsigned n) const { return (int)((uint64_t)(n >> 4) * mul >> shift); }
  __device__ __forceinline__ int part(int n) const { return n - whole(n) * size; }  // (n not negative)
  __device__ __forceinline__ int held(int tokens) const { return tokens > 0 ? whole((unsigned)tokens + size - 1) : 0; }
};

__device__ __forceinline__ int wave_total(int x) { return __builtin_amdgcn_readlane(wave_scan(x), 63); }

// Inclusive scans of N values a thread over the workgroup; `total` are the sums.  (Two barriers: what was in LDS before is
// written, and read, by then.)
template <int N> __device__ __forceinline__ void scan(int (&x)[N], int (*s_wave)[kThreads / 64], int (&total)[N]) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int n = 0; n < N; ++n) x[n] = wave_scan(x[n]);
  __syncthreads();
#pragma unroll
  for (int n = 0; n < N; ++n)
    if (lane == 63) s_wave[n][wave] = x[n];
  __syncthreads();
#pragma unroll
  for (int n = 0; n < N; ++n) {
    const int v = lane < kThreads / 64 ? s_wave[n][lane] : 0, upto = wave_scan(v);
    total[n] = __builtin_amdgcn_readlane(upto, kThreads / 64 - 1);
    x[n] += __builtin_amdgcn_readlane(upto, wave) - __builtin_amdgcn_readlane(v, wave);
  }
}
__device__ __forceinline__ int scan(int x, int (*s_wave)[kThreads / 64], int &total) {
  int y[1] = {x}, all[1];
  scan<1>(y, s_wave, all);
  total = all[0];
  return y[0];
}

// The maximum over the wave: rotations within rows of 16, then a lane of each.
template <int CTRL> __device__ __forceinline__ int rotated_max(int x) {
  return max(x, __builtin_amdgcn_update_dpp(x, x, CTRL, 0xf, 0xf, false));
}
__device__ __forceinline__ int max_of(int x) {
  x = rotated_max<0x121>(rotated_max<0x122>(rotated_max<0x124>(rotated_max<0x128>(x))));
  return max(max(__builtin_amdgcn_readlane(x, 0), __builtin_amdgcn_readlane(x, 16)),
             max(__builtin_amdgcn_readlane(x, 32), __builtin_amdgcn_readlane(x, 48)));
}
__device__ __forceinline__ int min_of(int x) { return ~max_of(~x); }

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
  int groups, beams;
  Page page;
  int blocks;           // of 64 columns
  unsigned by_beams;    // ceil(2^18 / beams): rows (below 2^13) by beams
  int ring;             // a power of two, no less than the rows
  int32_t *list_count;  // [groups * blocks]
  int32_t *list;        // [groups * blocks][beams * 64]
  int32_t *source;      // [groups * beams] the page that a row's copy comes from
};

// What becomes of a row, from its group's parents and lengths.
struct Row {
  int len;   // new
  int copy;  // the column of its own copy, -1: none
};
__device__ __forceinline__ Row row_of(int row, int parent, int parent_len, bool parent_stays, bool first, const Page &page, int width) {
  Row r{parent >= 0 ? max(parent_len, 0) : 0, -1};
  const bool keeps = parent_stays ? parent == row : first;
  const int last = page.whole(r.len);
  if (parent >= 0 && last * page.size != r.len && !keeps && last < width) r.copy = last;
  return r;
}

// One wave's 64 columns of a group; s_cells: [beams][64] of the wave, wave-uniform.  `free_page(page, where)` takes the
// lanes' pages that nobody holds any more, `source(row, page)` the page that a row's copy comes from.
//
// A row whose parent row r has n children: n - 1 more rows hold each full page of r, and its last page, where that is not
// full, one row or none.  So r's page in column c gains n - 1 holders, or loses one (the last page without children),
// whatever else holds it.  Where all rows hold one page the changes are added up first (a prefix: mostly nothing is
// left); elsewhere they go to page_shares one by one, gains before losses: the number of holders a group adds up to is
// then never below both its old and its new one, so the sum reaches -1 in one atomic only, the one after which no row of
// any group holds the page, whatever the order.
template <typename F, typename S>
__device__ __forceinline__ void follow_parents(const Reorder &p, int group, int block, int *s_cells, F free_page, S source) {
  const int lane = threadIdx.x & 63, beams = p.beams, c = block * 64 + lane;
  int *const mine = s_cells + lane;  // this lane's column: [beams], 64 apart
  // a lane a row
  const int known = min(lane, beams - 1), at = group * beams + known;
  const int old_len = max(p.lens[at], 0);
  int parent = p.parents[at];
  if (parent < 0 || parent >= beams) parent = -1;
  const int from = max(parent, 0);
  const int parent_len = __shfl(old_len, from), grandparent = __shfl(parent, from);  // (by every lane)
  // rows of the same parent, and this row's children, by the bits of the parents' numbers
  const bool alive = parent >= 0 && lane < beams;
  unsigned long long siblings = __ballot(alive), mine_of = siblings;
  for (int b = 0; 1 << b < beams; ++b) {
    const unsigned long long set = __ballot(parent >> b & 1);
    siblings &= parent >> b & 1 ? set : ~set;
    mine_of &= lane >> b & 1 ? set : ~set;
  }
  const bool first = lane == __builtin_ctzll(siblings | (unsigned long long)1 << 63);
  const int children = lane < beams ? __builtin_popcountll(mine_of) : 0;
  const Row row = row_of(known, parent, parent_len, parent >= 0 && grandparent == parent, first, p.page, p.width);
  const int held = min(p.page.held(old_len), p.width), new_held = min(p.page.held(row.len), p.width);
  const int partial = p.page.part(old_len) ? p.page.whole(old_len) : -1;  // the column of a last page that is not full
  const int most = max_of(lane < beams ? max(held, new_held) : 0);
  if (block * 64 >= most) return;  // nothing here
  int32_t *const cells = p.table + (int64_t)group * beams * p.t_sr + min(c, p.width - 1);
  // the cells, all rows' in flight together (of a lane behind the table: its last column; of rows that end before: whatever
  // lies there)
#pragma unroll 1
  for (int i = 0; i < beams; ++i)
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *)(cells + i * p.t_sr),
                                     (__attribute__((address_space(3))) void *)(s_cells + i * 64), 4, 0, 0);
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  const int page0 = mine[0];
  bool same = c < min_of(lane < beams ? held : INT32_MAX);  // all rows hold the page of row 0
#pragma unroll 4
  for (int i = 1; i < beams; ++i) same &= mine[i * 64] == page0;
  const bool settled = same;  // nothing of this column is written
  auto held_page = [&](int v) { return v >= 0 && v < p.pages; };
  // page_shares
  auto freed = [&](int v, bool gone) {
    if (gone) p.shares[v] = 0;
    free_page(v, __ballot(gone));
  };
  const unsigned long long rows = beams < 64 ? ((unsigned long long)1 << beams) - 1 : ~0ull;
  const unsigned long long gains = __ballot(children > 1) & rows, losses = __ballot(children == 0) & rows;
  if (gains | losses) {
    // rows whose last page is this column's count differently: no sum for it (nor where there is no page)
    unsigned long long ends = 0;
    for (unsigned long long m = __ballot(partial >= block * 64 && partial < block * 64 + 64) & rows; m;) {
      const int column = __builtin_amdgcn_readlane(partial, __builtin_ctzll(m));
      ends |= (unsigned long long)1 << (column - block * 64);
      m &= ~__ballot(partial == column);
    }
    same &= held_page(page0) && !(ends >> lane & 1);
    const int together = __builtin_popcountll(__ballot(parent >= 0) & rows) - beams;
    if (together != 0 && __ballot(same)) freed(page0, same && atomicAdd(p.shares + page0, together) + together == -1);
    if (__ballot(!same)) {
      if (gains) {
        for (unsigned long long m = gains; m;) {  // four at once
          int v[4], more[4];
#pragma unroll
          for (int i = 0; i < 4; ++i, m &= m - 1) {
            const int r = m ? __builtin_ctzll(m) : 0;
            v[i] = mine[r * 64];
            more[i] = m && c < __builtin_amdgcn_readlane(held, r) && c != __builtin_amdgcn_readlane(partial, r)
                          ? __builtin_amdgcn_readlane(children, r) - 1 : 0;
          }
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (!same && more[i] && held_page(v[i])) atomicAdd(p.shares + v[i], more[i]);
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // gains before losses
      }
      for (unsigned long long m = losses; m;) {  // eight at once
        int v[8], was[8];
#pragma unroll
        for (int i = 0; i < 8; ++i, m &= m - 1) {
          const int r = m ? __builtin_ctzll(m) : 0;
          v[i] = mine[r * 64];
          was[i] = 1;
          if (m && !same && c < __builtin_amdgcn_readlane(held, r) && held_page(v[i])) was[i] = atomicAdd(p.shares + v[i], -1);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (__ballot(was[i] == 0)) freed(v[i], was[i] == 0);
      }
    }
  }
  // a lane a row: where its copy comes from, and the columns that it is given
  int upto = alive && !(parent == lane && row.copy < 0) ? new_held : 0;  // (else given up, or as it was)
  if (lane < beams && row.copy >= block * 64 && row.copy < block * 64 + 64) {
    const int v = s_cells[from * 64 + row.copy - block * 64];
    source(group * beams + lane, v);
    if (held_page(v)) upto = row.copy;  // (its own page comes from the pool)
  }
  if (!__ballot(!settled)) return;
  int32_t *to = cells;
  for (int i0 = 0; i0 < beams; i0 += 4) {
    int v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = mine[__builtin_amdgcn_readlane(from, i0 + i) * 64];  // (rows behind the last: upto 0)
#pragma unroll
    for (int i = 0; i < 4; ++i, to += p.t_sr)
      if (!settled && c < __builtin_amdgcn_readlane(upto, i0 + i)) *to = v[i];
  }
}

// LDS of share_out, in ints: the bitmap, list offsets, then lengths, parents and (`ring`) the freed pages that are on top.
__host__ __device__ constexpr int bitmap_words(int pages) { return ((pages < kBitmap ? pages : kBitmap) + 31) / 32; }
__host__ __device__ constexpr int pool_ints(int pages, int units, int rows, int ring) {
  return bitmap_words(pages) + (units < kUnits ? units : kUnits) + 1 + 2 * rows + ring;
}

// The pool, one workgroup: freed pages onto the stack by number, then each row's copy from it.  The pages to take are the
// last that were freed, or lie where nothing is written: nothing is read back.  `marked`: the freed pages are in the
// bitmap already, else in lists a wave.  PER: rows a thread, at most: 1, or all that there may be (256 rows 13.9 and 14.5 us
// a call).
template <int PER> __device__ __forceinline__ void share_out(const Reorder &p, int *s_mem, int (*s_wave)[kThreads / 64], bool marked,
                                          const int *s_source) {
  const int tid = threadIdx.x, rows = p.groups * p.beams, units = p.groups * p.blocks;
  unsigned int *const s_bits = (unsigned int *)s_mem;
  int *const s_at = s_mem + bitmap_words(p.pages), *const s_len = s_at + min(units, kUnits) + 1;
  int *const s_parent = s_len + rows, *const s_top = s_parent + rows, *const s_first = s_top;  // (done with by then)
  const int count = min(max(*p.count, 0), p.pool);
  __shared__ int s_short;  // a row found no page
  if (tid == 0) s_short = 0;
#pragma unroll 1
  for (int r = tid; r < rows; r += kThreads) {
    s_len[r] = p.lens[r];
    s_parent[r] = p.parents[r];
    s_first[r] = L20_PD_MAX_BEAMS;
  }
  constexpr int kLists = kUnits / kThreads;
  int lengths[kLists];  // of the first kUnits lists
#pragma unroll
  for (int i = 0; i < kLists; ++i) {
    const int u = tid * kLists + i;
    lengths[i] = !marked && u < units ? p.list_count[u] : 0;
  }
  const int per_row = PER == 1 ? 1 : (rows + kThreads - 1) / kThreads;
  int from[PER];  // (of rows without a copy: whatever is there)
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int r = tid * per_row + i;
    if (i < per_row && r < rows) from[i] = s_source ? s_source[r] : p.source[r];
  }
  // rows that need a page, in order
  Row row[PER];
  int wanted = 0;
  __syncthreads();
  auto row_at = [&](int r, int &me, int &parent) {  // its group's first row
    const int base = (int)((unsigned)r * p.by_beams >> 18) * p.beams;
    me = r - base;
    parent = s_parent[r];
    if (parent < 0 || parent >= p.beams) parent = -1;
    return base;
  };
#pragma unroll 1
  for (int r = tid; r < rows; r += kThreads) {
    int me, parent;
    const int base = row_at(r, me, parent);
    if (parent >= 0) atomicMin(s_first + base + parent, me);
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int r = tid * per_row + i;
    row[i] = Row{0, -1};
    if (i < per_row && r < rows) {
      int me, parent;
      const int base = row_at(r, me, parent), from_row = base + max(parent, 0);
      row[i] = row_of(me, parent, s_len[from_row], parent >= 0 && s_parent[from_row] == parent, s_first[from_row] == me, p.page,
                      p.width);
      if (row[i].copy >= 0 && (from[i] < 0 || from[i] >= p.pages)) row[i].copy = -1;  // the parent has no page there either
      wanted += row[i].copy >= 0;
    }
  }
  int upto[2] = {wanted, 0}, totals[2];
#pragma unroll
  for (int i = 0; i < kLists; ++i) upto[1] += lengths[i];
  const int listed = upto[1];
  scan<2>(upto, s_wave, totals);
  const int total = totals[0], first_wanted = upto[0] - wanted;
  // freed pages, by number; places from the top are known once all are counted
  int freed = 0;
  auto push = [&](int base, int words) {
    const int per = (words + kThreads - 1) / kThreads;
    int mine = 0;
#pragma unroll 1
    for (int i = 0; i < per; ++i)
      if (tid * per + i < words) mine += __builtin_popcount(s_bits[tid * per + i]);
    int here;
    int rank = freed + scan(mine, s_wave, here) - mine;
    const int last = min(freed + here, p.pool - count);  // (`rows` of these: a place each)
    for (int i = 0; i < per && tid * per + i < words; ++i)
      for (unsigned int w = s_bits[tid * per + i]; w; w &= w - 1, ++rank) {
        const int page = base + (tid * per + i) * 32 + __builtin_ctz(w);
        if (rank >= last) continue;
        p.stack[count + rank] = page;
        if (rank >= last - rows) s_top[rank & (p.ring - 1)] = page;
      }
    freed += here;
    __syncthreads();
  };
  if (marked) {
    push(0, bitmap_words(p.pages));
  } else {
    for (int base = 0; base < p.pages; base += kBitmap) {
      const int n = min(p.pages - base, kBitmap), words = (n + 31) / 32;
      for (int i = tid; i < words; i += kThreads) s_bits[i] = 0;
      bool some = false;
      for (int u0 = 0; u0 < units; u0 += kUnits) {  // the entries of kUnits lists, spread over the threads
        const int here = min(units - u0, kUnits);
        int mine = 0, length[kLists];
#pragma unroll
        for (int i = 0; i < kLists; ++i) {
          const int u = u0 + tid * kLists + i;
          length[i] = u0 == 0 ? lengths[i] : u < units ? p.list_count[u] : 0;
          mine += length[i];
        }
        int entries = totals[1], at = upto[1] - listed;
        if (base > 0 || u0 > 0) at = scan(mine, s_wave, entries) - mine;
        else __syncthreads();  // the bitmap is clear; offsets of other lists are read
        if (entries == 0) continue;
        some = true;
#pragma unroll
        for (int i = 0; i < kLists; ++i) {
          if (tid * kLists + i < here) s_at[tid * kLists + i] = at;
          at += length[i];
        }
        __syncthreads();
        for (int k = tid; k < entries; k += kThreads) {
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
      push(base, words);
    }
  }
  const int have = (int)min((int64_t)count + freed, (int64_t)p.pool), kept = have - count;
  int got[PER], served = 0, k = first_wanted;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int r = tid * per_row + i;
    got[i] = -1;
    if (i < per_row && r < rows) {
      p.lens[r] = row[i].len;
      if (row[i].copy >= 0) {
        if (k < have) got[i] = k < kept ? s_top[(kept - 1 - k) & (p.ring - 1)] : p.stack[have - 1 - k];
        ++k;
        if (got[i] < 0 || got[i] >= p.pages) got[i] = -1;
        p.table[r * p.t_sr + row[i].copy] = got[i];
        served += got[i] >= 0;
      }
    }
  }
  int pairs = total, at = first_wanted;
  if (served != wanted) s_short = 1;
  __syncthreads();
  if (s_short) at = scan(served, s_wave, pairs) - served;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    if (got[i] >= 0) {
      p.src[at] = from[i];
      p.dst[at] = got[i];
      p.tokens[at] = p.page.part(row[i].len);
      ++at;
    }
  }
#pragma unroll 1
  for (int i = pairs + tid; i < p.room; i += kThreads) p.src[i] = -1, p.dst[i] = -1, p.tokens[i] = 0;
  if (tid == 0) {
    p.pairs[0] = pairs;
    p.pairs[1] = total - pairs;
    *p.count = have - min(total, have);
  }
}

__global__ __launch_bounds__(64 * kCellWaves) void rp_cells(Reorder p) {
  extern __shared__ int s_mem[];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int group = blockIdx.y, block = blockIdx.x * kCellWaves + wave;
  if (block >= p.blocks) return;
  const int unit = group * p.blocks + block;
  int32_t *const list = p.list + (int64_t)unit * p.beams * 64;
  int listed = 0;
  follow_parents(
      p, group, block, s_mem + wave * p.beams * 64,
      [&](int v, unsigned long long which) {
        if (which >> lane & 1) list[listed + __builtin_popcountll(which & (((unsigned long long)1 << lane) - 1))] = v;
        listed += __builtin_popcountll(which);
      },
      [&](int row, int v) { p.source[row] = v; });
  if (lane == 0) p.list_count[unit] = listed;
}

template <int PER> __global__ __launch_bounds__(kThreads) void rp_pool(Reorder p) {
  extern __shared__ int s_mem[];
  __shared__ int s_wave[2][kThreads / 64];
  share_out<PER>(p, s_mem, s_wave, false, nullptr);
}

// Both in one launch, for few waves' worth of cells: freed pages go straight into the bitmap.
__global__ __launch_bounds__(kThreads) void rp_small(Reorder p) {
  extern __shared__ int s_mem[];
  __shared__ int s_wave[2][kThreads / 64];
  __shared__ int s_source[kSmall * L20_PD_MAX_BEAMS];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int units = p.groups * p.blocks, words = bitmap_words(p.pages);
  int *const s_cells = s_mem + pool_ints(p.pages, units, p.groups * p.beams, p.ring);
#pragma unroll 1
  for (int i = threadIdx.x; i < words; i += kThreads) s_mem[i] = 0;
  __syncthreads();
#pragma unroll 1
  for (int unit = wave; unit < units; unit += kThreads / 64) {
    const int group = unit / p.blocks;
    follow_parents(
        p, group, unit - group * p.blocks, s_cells + wave * p.beams * 64,
        [&](int v, unsigned long long which) {
          if (which >> lane & 1) atomicOr((unsigned int *)s_mem + (v >> 5), 1u << (v & 31));
        },
        [&](int row, int v) { s_source[row] = v; });
  }
  __syncthreads();
  static_assert(kSmall * L20_PD_MAX_BEAMS <= kThreads, "a row a thread");
  share_out<1>(p, s_mem, s_wave, true, s_source);
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
  int rows;
  Page page;
  int words;           // of a bitmap of the pages
  unsigned int *high;  // pages held at or beyond the limit
  unsigned int *low;   // free ones below it
  int32_t *rank;       // [words] set bits of `high` before a word
  int row_blocks;      // of 256 columns, a row
};

// Bits of both bitmaps before word `first`, and of all, by the workgroup: every one counts for itself, 8 bytes a 32 pages.
template <int THREADS>
__device__ __forceinline__ void bits_before(const unsigned int *high, const unsigned int *low, int words, int first, int (*s_sum)[THREADS / 64],
                                            int (&before)[2], int (&all)[2]) {
  int n[4] = {0, 0, 0, 0};
  for (int i0 = threadIdx.x; i0 < words; i0 += 8 * THREADS) {  // eight loads of each at once
    unsigned int h[8], l[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const int i = i0 + u * THREADS;
      h[u] = i < words ? high[i] : 0;
      l[u] = i < words ? low[i] : 0;
    }
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const bool below = i0 + u * THREADS < first;
      n[0] += below ? __builtin_popcount(h[u]) : 0;
      n[1] += below ? __builtin_popcount(l[u]) : 0;
      n[2] += __builtin_popcount(h[u]);
      n[3] += __builtin_popcount(l[u]);
    }
  }
#pragma unroll
  for (int k = 0; k < 4; ++k) n[k] = wave_total(n[k]);
  if ((threadIdx.x & 63) == 0)
#pragma unroll
    for (int k = 0; k < 4; ++k) s_sum[k][threadIdx.x >> 6] = n[k];
  __syncthreads();
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    before[k] = wave_total(lane < THREADS / 64 ? s_sum[k][lane] : 0);
    all[k] = wave_total(lane < THREADS / 64 ? s_sum[2 + k][lane] : 0);
  }
}

// A page to its place, by its rank in its bitmap (a lane a page: neighbours store side by side): src or dst, or, what
// stays free, the stack (the lowest on top).
__device__ __forceinline__ void place(const Compact &p, int page, bool high, bool low, int at_high, int at_low, int moves, int all_low) {
  if (high && at_high < moves) p.src[at_high] = page;
  if (low) {
    if (at_low < moves) p.dst[at_low] = page;
    else if (all_low - 1 - at_low < p.pool) p.stack[all_low - 1 - at_low] = page;
  }
}
// What goes with pair k, and what stands behind the pairs.
__device__ __forceinline__ void settle_pair(const Compact &p, int k, int moves) {
  if (k < moves) {
    const int from = p.src[k], to = p.dst[k];
    p.shares[to] = p.shares[from];
    p.shares[from] = 0;
    p.tokens[k] = p.page.size;
  } else {
    p.src[k] = -1, p.dst[k] = -1, p.tokens[k] = 0;
  }
}
__device__ __forceinline__ void finish(const Compact &p, int moves, int all_high, int all_low) {
  *p.count = all_low - moves;
  p.pairs[0] = moves;
  p.pairs[1] = all_high - moves;
}

__global__ __launch_bounds__(256) void cp_clear(Compact p) {
  const int i = blockIdx.x * 256 + threadIdx.x;
  if (i < p.words) p.high[i] = p.low[i] = 0;
}

__global__ __launch_bounds__(256) void cp_mark(Compact p) {
  const int64_t tables = (int64_t)p.rows * p.row_blocks;
  if (blockIdx.x < tables) {
    const int row = (int)(blockIdx.x / p.row_blocks), c = (int)(blockIdx.x % p.row_blocks) * 256 + threadIdx.x;
    if (c >= min(p.page.held(p.lens[row]), p.width)) return;
    const int v = p.table[row * p.t_sr + c];
    if (v >= p.limit && v < p.pages) atomicOr(p.high + (v >> 5), 1u << (v & 31));
  } else {
    const int64_t i = (blockIdx.x - tables) * 256 + threadIdx.x;
    if (i >= min(max(*p.count, 0), p.pool)) return;
    const int v = p.stack[i];
    if (v >= 0 && v < p.limit) atomicOr(p.low + (v >> 5), 1u << (v & 31));
  }
}

// A thread `each` pages, kThreads apart: a workgroup a CU at most, since every one counts all pages (a call with
// one page a thread and so: 2^20 pages 76 and 68 us, 2^24 6.0 and 0.73 ms).
__global__ __launch_bounds__(kThreads) void cp_place(Compact p, int each) {
  constexpr int kWaves = kThreads / 64;
  __shared__ int s_sum[4][kWaves], s_wave[2][2][kWaves];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t first = (int64_t)blockIdx.x * each * kThreads;
  int before[2], all[2], moves = 0;
  for (int i = 0; i < each; ++i) {
    const int64_t page = first + (int64_t)i * kThreads + threadIdx.x;
    if (page - threadIdx.x >= p.pages) break;
    const int word = (int)(page >> 5), bit = (int)(page & 31);
    const unsigned int h = word < p.words ? p.high[word] : 0, l = word < p.words ? p.low[word] : 0;
    const bool high = h >> bit & 1, low = l >> bit & 1;
    const unsigned long long highs = __ballot(high), lows = __ballot(low), below = ((unsigned long long)1 << lane) - 1;
    int (*const s_here)[kWaves] = s_wave[i & 1];
    if (lane == 0) s_here[0][wave] = __builtin_popcountll(highs), s_here[1][wave] = __builtin_popcountll(lows);
    if (i == 0) {
      bits_before<kThreads>(p.high, p.low, p.words, (int)(first >> 5), s_sum, before, all);  // (its barrier)
      moves = min(min(all[0], all[1]), p.room);
    } else {
      __syncthreads();
    }
    int at[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int n = lane < kWaves ? s_here[k][lane] : 0;
      at[k] = before[k] + wave_total(lane < wave ? n : 0);
      before[k] += wave_total(n);
    }
    at[0] += __builtin_popcountll(highs & below), at[1] += __builtin_popcountll(lows & below);
    if (bit == 0 && word < p.words) p.rank[word] = at[0];
    place(p, (int)page, high, low, at[0], at[1], moves, all[1]);
    if (page == 0) finish(p, moves, all[0], all[1]);
  }
}

// Where the page of a cell goes: its rank among the pages to move says which pair.
__device__ __forceinline__ void remap(const Compact &p, const unsigned int *high, const int *rank, int row, int c, int moves) {
  if (c >= min(p.page.held(p.lens[row]), p.width)) return;
  int32_t *const cell = p.table + row * p.t_sr + c;
  const int v = *cell;
  if (v < p.limit || v >= p.pages) return;
  const int k = rank[v >> 5] + __builtin_popcount(high[v >> 5] & ((1u << (v & 31)) - 1));
  if (k < moves) *cell = p.dst[k];
}

__global__ __launch_bounds__(256) void cp_remap(Compact p) {
  const int64_t tables = (int64_t)p.rows * p.row_blocks;
  const int moves = p.pairs[0];
  if (blockIdx.x < tables) {
    remap(p, p.high, p.rank, (int)(blockIdx.x / p.row_blocks), (int)(blockIdx.x % p.row_blocks) * 256 + threadIdx.x, moves);
  } else {
    const int64_t k = (blockIdx.x - tables) * 256 + threadIdx.x;
    if (k < p.room) settle_pair(p, (int)k, moves);
  }
}

// All of it in one workgroup, the bitmaps in LDS.
__global__ __launch_bounds__(kThreads) void cp_small(Compact p) {
  __shared__ unsigned int s_high[kSmallPages / 32], s_low[kSmallPages / 32];
  __shared__ int s_rank[kSmallPages / 32], s_rank_low[kSmallPages / 32], s_wave[2][kThreads / 64];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int count = min(max(*p.count, 0), p.pool);
  for (int i = tid; i < p.words; i += kThreads) s_high[i] = s_low[i] = 0;
  __syncthreads();
  for (int i = tid; i < count; i += kThreads) {
    const int v = p.stack[i];
    if (v >= 0 && v < p.limit) atomicOr(s_low + (v >> 5), 1u << (v & 31));
  }
  for (int row = wave; row < p.rows; row += kThreads / 64) {
    const int held = min(p.page.held(p.lens[row]), p.width);
    for (int c = lane; c < held; c += 64) {
      const int v = p.table[row * p.t_sr + c];
      if (v >= p.limit && v < p.pages) atomicOr(s_high + (v >> 5), 1u << (v & 31));
    }
  }
  __syncthreads();
  static_assert(kSmallPages / 32 <= kThreads, "a word a thread");
  const int bits[2] = {tid < p.words ? __builtin_popcount(s_high[tid]) : 0, tid < p.words ? __builtin_popcount(s_low[tid]) : 0};
  int upto[2] = {bits[0], bits[1]}, all[2];
  scan<2>(upto, s_wave, all);
  const int all_high = all[0], all_low = all[1], moves = min(min(all_high, all_low), p.room);
  if (tid < p.words) s_rank[tid] = upto[0] - bits[0], s_rank_low[tid] = upto[1] - bits[1];
  __syncthreads();
  for (int page = tid; page < p.pages; page += kThreads) {
    const unsigned int h = s_high[page >> 5], l = s_low[page >> 5], bit = 1u << (page & 31);
    place(p, page, h & bit, l & bit, s_rank[page >> 5] + __builtin_popcount(h & (bit - 1)),
          s_rank_low[page >> 5] + __builtin_popcount(l & (bit - 1)), moves, all_low);
  }
  __syncthreads();
  for (int k = tid; k < p.room; k += kThreads) settle_pair(p, k, moves);
  for (int row = wave; row < p.rows; row += kThreads / 64) {
    const int held = min(p.page.held(p.lens[row]), p.width);
    for (int c = lane; c < held; c += 64) remap(p, s_high, s_rank, row, c, moves);
  }
  if (tid == 0) finish(p, moves, all_high, all_low);
}

constexpr int kCaches = 64;  // caches of a launch
// Bytes of a run from which on a workgroup takes it by itself.  Measured, 512 pages of 16 caches by runs and by divisions:
// whole pages with runs of 2 KB 42.5 and 21.1 us, 4 KB 63.5 and 48.1, 8 KB 113.9 and 113.7, 16 KB 218 and 218; half of their
// tokens, 8 KB 66.9 and 60.8, 16 KB 119 and 125, 32 KB 271 and 283.
constexpr int kRun = 16384;

struct Copy {
  const int32_t *src, *dst, *tokens;
  int room;
  const int32_t *count;
  char *cache[kCaches];
  int caches;
  int64_t pages, page_stride;
  // A page is `runs` runs of bytes, of which the first tokens are the first bytes (`token_bytes` each; 0: whole) ...
  int runs;
  int64_t run_stride, token_bytes;
  // ... or any three levels, outside in, above `inner` contiguous bytes.
  uint32_t size[3];
  int64_t stride[3];
  uint32_t inner;  // units
  int token_level;
  int64_t units;    // of a run (of a page), each sizeof(V) bytes
  int64_t segment;  // units a workgroup takes at once
  int segments;     // of a run (of a page)
};

template <typename V, bool RUNS> __global__ __launch_bounds__(256) void pc_copy(Copy p) {
  const int pairs = p.count ? min(max(*p.count, 0), p.room) : p.room;
  const int64_t all = (int64_t)pairs * p.caches * p.runs * p.segments;
  for (int64_t job = blockIdx.x; job < all; job += gridDim.x) {
    int64_t rest = job / p.segments;
    const int segment = (int)(job - rest * p.segments), run = (int)(rest % p.runs);
    rest /= p.runs;
    const int cache = (int)(rest % p.caches), pair = (int)(rest / p.caches);
    const int from = p.src[pair], to = p.dst[pair];
    if (from < 0 || from >= p.pages || to < 0 || to >= p.pages) continue;
    const int tokens = p.tokens ? max(p.tokens[pair], 0) : INT32_MAX;
    const char *const a = p.cache[cache] + from * p.page_stride;
    char *const b = p.cache[cache] + to * p.page_stride;
    const int64_t first = segment * p.segment + threadIdx.x;
    int64_t end = min(((int64_t)segment + 1) * p.segment, p.units);
    if constexpr (RUNS) {
      const V *const x = reinterpret_cast<const V *>(a + run * p.run_stride);
      V *const y = reinterpret_cast<V *>(b + run * p.run_stride);
      if (p.token_bytes) {
        const int64_t bytes = tokens * p.token_bytes, whole = bytes / (int64_t)sizeof(V);
        if (whole < end) {  // the tokens end here, or before
          end = whole;
          const int odd = (int)(bytes - whole * (int64_t)sizeof(V));  // inside a unit
          if (whole >= segment * p.segment && (int)threadIdx.x < odd)
            reinterpret_cast<char *>(y + whole)[threadIdx.x] = reinterpret_cast<const char *>(x + whole)[threadIdx.x];
        }
      }
      for (int64_t i = first; i < end; i += 4 * 256) {
        V v[4];
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (i + j * 256 < end) v[j] = x[i + j * 256];
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (i + j * 256 < end) y[i + j * 256] = v[j];
      }
    } else {
      for (int64_t i = first; i < end; i += 256) {
        const uint32_t n = (uint32_t)i, x = n / p.inner, y = x / p.size[2], x0 = y / p.size[1];
        const uint32_t x2 = x - y * p.size[2], x1 = y - x0 * p.size[1];
        const uint32_t token = p.token_level == 0 ? x0 : p.token_level == 1 ? x1 : p.token_level == 2 ? x2 : 0;
        if (p.token_level >= 0 && token >= (uint32_t)tokens) continue;
        const int64_t at = x0 * p.stride[0] + x1 * p.stride[1] + x2 * p.stride[2] + (n - x * p.inner) * (int64_t)sizeof(V);
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
  constexpr int64_t kFar = (int64_t)1 << 40;  // no level reaches further: sums and products of these stay within 64 bits
  const auto far = [](int64_t n, int64_t step) { return n > kMaxCells || (n > 1 && step > kFar / (n - 1)); };
  int64_t bytes = a->inner, span[4] = {a->inner, a->inner, a->inner, a->inner};  // of a step of the level inside
  for (int i = 2; i >= 0; --i) {
    if (bytes > INT32_MAX || far(size[i], stride[i])) return set_error(L20_PD_EINVAL, "page too large");
    if (size[i] > 1 && stride[i] < span[i + 1]) return set_error(L20_PD_EINVAL, "a page's parts overlap");
    span[i] = (size[i] > 1 ? (size[i] - 1) * stride[i] : 0) + span[i + 1];
    bytes *= size[i];
  }
  if (bytes > INT32_MAX) return set_error(L20_PD_EINVAL, "page too large");
  if (a->pages > 1) {  // pages are a level among the others, wherever their stride puts them
    if (far(a->pages, a->stride_page)) return set_error(L20_PD_EINVAL, "cache too large");
    if (a->stride_page < 1) return set_error(L20_PD_EINVAL, "pages overlap");
    int64_t inside = a->inner;
    bool placed = false;
    for (int i = 2; i >= -1; --i) {
      if (!placed && (i < 0 || (size[i] > 1 && stride[i] > a->stride_page))) {
        if (a->stride_page < inside) return set_error(L20_PD_EINVAL, "pages overlap");
        inside += (a->pages - 1) * a->stride_page;
        placed = true;
      }
      if (i < 0 || size[i] == 1) continue;
      if (stride[i] < inside) return set_error(L20_PD_EINVAL, "pages overlap");
      inside += (size[i] - 1) * stride[i];
    }
  }
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

// Every tensor of these calls is read or written throughout: none may share bytes with another.
template <typename A> int32_t apart(const A *a, const void *parents, int64_t rows, int64_t workspace_bytes) {
  using l20la::Lattice;
  const auto run = [](const void *at, int64_t bytes) { return Lattice(at, 0, 0, bytes > 0 ? 1 : 0, 1, bytes); };
  const Lattice all[] = {Lattice(a->block_table, a->bt_stride_row * 4, 0, rows, 1, (int64_t)a->table_pages * 4),
                         run(a->seq_lens, rows * 4),
                         run(a->page_shares, (int64_t)a->pages * 4),
                         run(a->free_pages, (int64_t)a->pool * 4),
                         run(a->free_count, 4),
                         run(a->src, (int64_t)a->room * 4),
                         run(a->dst, (int64_t)a->room * 4),
                         run(a->tokens, (int64_t)a->room * 4),
                         run(a->count, 8),
                         run(a->workspace, workspace_bytes),
                         run(parents, parents ? rows * 4 : 0)};
  constexpr int n = sizeof(all) / sizeof(all[0]);
  for (int i = 0; i < n; ++i)
    for (int j = 0; j < i; ++j)
      if (l20la::overlap(all[i], all[j])) return set_error(L20_PD_EINVAL, "tensors and workspace must lie apart");
  return L20_PD_OK;
}

template <int PER> int32_t launch_pool(const l20pm::Reorder &p, int most, int lds, hipStream_t s) {
  static l20la::LdsLimit limit;
  const hipError_t e = limit.raise(reinterpret_cast<const void *>(&l20pm::rp_pool<PER>), most);
  if (e != hipSuccess) return set_error(L20_PD_ELAUNCH, hipGetErrorString(e));
  hipLaunchKernelGGL(l20pm::rp_pool<PER>, dim3(1), dim3(l20pm::kThreads), (size_t)lds, s, p);
  return launched();
}

template <typename V> int32_t launch_copy(const l20pm::Copy &p, bool runs, hipStream_t s) {
  const int64_t jobs = (int64_t)p.room * p.caches * p.runs * p.segments;
  const unsigned grid = (unsigned)std::min<int64_t>(jobs, 8 * (int64_t)l20la::device_cus());
  if (runs) hipLaunchKernelGGL((l20pm::pc_copy<V, true>), dim3(grid), dim3(256), 0, s, p);
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
  rc = apart(a, a->parents, (int64_t)a->groups * a->beams, a->groups > 0 ? workspace(a) : 0);
  if (rc != L20_PD_OK) return rc;
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
  p.page = l20pm::Page(a->page_size);
  p.blocks = a->groups > 0 ? (a->table_pages + 63) / 64 : 0;
  p.list_count = reinterpret_cast<int32_t *>(a->workspace);
  p.list = p.list_count + (int64_t)p.groups * p.blocks;
  p.source = p.list + (int64_t)p.groups * p.blocks * p.beams * 64;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const int rows = p.groups * p.beams, units = p.groups * p.blocks;
  p.by_beams = ((1u << 18) + p.beams - 1) / p.beams;
  for (p.ring = 1; p.ring < rows;) p.ring *= 2;
  const int most = 4 * l20pm::pool_ints(l20pm::kBitmap, l20pm::kUnits, L20_PD_MAX_REQUESTS, L20_PD_MAX_REQUESTS);
  const int lds = 4 * l20pm::pool_ints(p.pages, units, rows, p.ring), cells = l20pm::kThreads / 64 * p.beams * 256;
  if (units <= l20pm::kSmall && p.pages <= l20pm::kBitmap && lds + cells <= most) {
    static l20la::LdsLimit limit;
    const hipError_t e = limit.raise(reinterpret_cast<const void *>(&l20pm::rp_small), most);
    if (e != hipSuccess) return set_error(L20_PD_ELAUNCH, hipGetErrorString(e));
    hipLaunchKernelGGL(l20pm::rp_small, dim3(1), dim3(l20pm::kThreads), (size_t)(lds + cells), s, p);
    return launched();
  }
  if (units > 0) {  // (without groups the pool's part alone: it says that there is nothing to copy)
    const dim3 grid((unsigned)((p.blocks + l20pm::kCellWaves - 1) / l20pm::kCellWaves), (unsigned)p.groups);
    hipLaunchKernelGGL(l20pm::rp_cells, grid, dim3(64 * l20pm::kCellWaves), (size_t)l20pm::kCellWaves * p.beams * 256, s, p);
    rc = launched();
    if (rc != L20_PD_OK) return rc;
  }
  return rows <= l20pm::kThreads ? launch_pool<1>(p, most, lds, s) : launch_pool<l20pm::kPerThread>(p, most, lds, s);
}

int32_t l20_pd_compact_pages_check(const l20_pd_compact_args *a) {
  l20pd_host::clear_error();
  return check(a);
}

int64_t l20_pd_compact_pages_workspace(const l20_pd_compact_args *a) {
  return a && a->pages > 0 ? 12 * words_of(a) : 0;
}

int32_t l20_pd_compact_pages(const l20_pd_compact_args *a, void *stream) {
  l20pd_host::clear_error();
  int32_t rc = check(a);
  if (rc != L20_PD_OK) return rc;
  if (!a->workspace || (uintptr_t)a->workspace % 4 || a->workspace_bytes < l20_pd_compact_pages_workspace(a))
    return set_error(L20_PD_EINVAL, "workspace is missing, misaligned or too small");
  rc = apart(a, nullptr, a->rows, l20_pd_compact_pages_workspace(a));
  if (rc != L20_PD_OK) return rc;
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
  p.page = l20pm::Page(a->page_size);
  p.words = (int)words_of(a);
  p.high = reinterpret_cast<unsigned int *>(a->workspace);
  p.low = p.high + p.words;
  p.rank = reinterpret_cast<int32_t *>(p.low + p.words);
  p.row_blocks = std::max(1, (a->table_pages + 255) / 256);
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  if (p.pages <= l20pm::kSmallPages && (int64_t)p.rows * ((p.width + 63) / 64) <= l20pm::kSmallWaves) {
    hipLaunchKernelGGL(l20pm::cp_small, dim3(1), dim3(l20pm::kThreads), 0, s, p);
    return launched();
  }
  const auto blocks = [](int64_t n) { return (unsigned)((n + 255) / 256); };
  const unsigned tables = (unsigned)(p.rows * (int64_t)p.row_blocks);
  hipLaunchKernelGGL(l20pm::cp_clear, dim3(blocks(p.words)), dim3(256), 0, s, p);
  hipLaunchKernelGGL(l20pm::cp_mark, dim3(tables + blocks(p.pool)), dim3(256), 0, s, p);
  const int chunks = (p.pages + l20pm::kThreads - 1) / l20pm::kThreads, cus = l20la::device_cus(), each = (chunks + cus - 1) / cus;
  hipLaunchKernelGGL(l20pm::cp_place, dim3((unsigned)((chunks + each - 1) / each)), dim3(l20pm::kThreads), 0, s, p, each);
  if (tables + blocks(p.room) > 0) hipLaunchKernelGGL(l20pm::cp_remap, dim3(tables + blocks(p.room)), dim3(256), 0, s, p);
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
  p.token_level = a->tokens ? a->token_level : -1;
  if (p.token_level < 0) p.tokens = nullptr;
  const int64_t size[3] = {a->size0, a->size1, a->size2};
  int64_t stride[3] = {a->stride0, a->stride1, a->stride2}, dense[4];  // dense[i]: bytes of one step of level i - 1, if dense
  dense[3] = a->inner;
  uint64_t low = (uint64_t)p.page_stride;  // what every address is a multiple of
  for (int i = 0; i < a->num_caches; ++i) low |= (uint64_t)(uintptr_t)a->caches[i];
  uint64_t steps = (uint64_t)a->inner;
  for (int i = 2; i >= 0; --i) {
    if (size[i] == 1) stride[i] = dense[i + 1];  // (of one step: as if dense)
    else steps |= (uint64_t)stride[i];
    dense[i] = size[i] * dense[i + 1];
  }
  // One run a step of level 0, or one in all: what is below is dense, and its tokens, if they are counted, outside.
  const bool below = stride[1] == dense[2] && stride[2] == dense[3];
  const bool one = below && stride[0] == dense[1] && p.token_level <= 0;
  const bool runs = one || (below && (p.token_level < 0 || p.token_level == 1) && dense[1] >= l20pm::kRun);
  p.runs = runs && !one ? (int)size[0] : 1;
  p.run_stride = stride[0];
  p.token_bytes = p.token_level < 0 ? 0 : stride[p.token_level];
  const int64_t bytes = runs && !one ? dense[1] : dense[0];
  low |= !runs ? steps : one ? (uint64_t)bytes : (uint64_t)bytes | (uint64_t)stride[0];
  const int unit = low % 16 == 0 ? 16 : low % 8 == 0 ? 8 : low % 4 == 0 ? 4 : low % 2 == 0 ? 2 : 1;
  for (int i = 0; i < 3; ++i) p.size[i] = (uint32_t)size[i], p.stride[i] = stride[i];
  p.inner = (uint32_t)(a->inner / unit);
  p.units = bytes / unit;
  p.segment = std::min<int64_t>(p.units, 1024);
  p.segments = (int)((p.units + p.segment - 1) / p.segment);
  for (int first = 0; first < a->num_caches && rc == L20_PD_OK; first += l20pm::kCaches) {
    p.caches = std::min(l20pm::kCaches, a->num_caches - first);
    for (int i = 0; i < p.caches; ++i) p.cache[i] = reinterpret_cast<char *>(a->caches[first + i]);
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    rc = unit == 16  ? launch_copy<l20la::i32x4>(p, runs, s)
         : unit == 8 ? launch_copy<l20la::i32x2>(p, runs, s)
         : unit == 4 ? launch_copy<int32_t>(p, runs, s)
         : unit == 2 ? launch_copy<int16_t>(p, runs, s)
                     : launch_copy<int8_t>(p, runs, s);
  }
  return rc;
}

}  // extern "C"
