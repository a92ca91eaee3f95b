/*
 * C ABI of the block tables and the page pool in libl20_paged_decode_hip.so, on the GPU: a batch's block tables,
 * slot map, positions and lengths from its request lengths; rows that follow their parents (forks, copies on
 * write, pages given back); the pool's compaction; and the copies of pages that these ask for.  Return codes and
 * l20_pd_last_error() are those of l20_paged_decode.h.  The reference's callers do this on the host: no
 * counterpart there.
 */
#ifndef L20_BLOCK_TABLES_H_
#define L20_BLOCK_TABLES_H_

#include <stdint.h>

#include "l20_paged_decode.h"

#ifdef __cplusplus
extern "C" {
#endif

#define L20_PD_MAX_REQUESTS 8192

/*
 *   cached_lens [batch] int32: tokens in the cache (below 0: none)
 *   new_lens    [batch] int32: tokens to append; below 0: the request is finished
 *   block_table [batch, table_pages] int32, updated: request b holds its first
 *               ceil(cached_lens[b] / page_size) cells
 *   free_pages  [pool] int32 stack, updated: cells 0 .. free_count - 1 are free page ids
 *   free_count  [1] int32, free_count_out [1] int32 (may be the same memory)
 *   slots, positions [num_slots] int64; cu_lens [batch + 1] int32; seq_lens [batch] int32 (outputs)
 *
 * In this order: the pages of finished requests go on top of the stack (request by request, a row's
 * cells in order; what the stack cannot hold is dropped).  Then the requests are served in order, each
 * taking the pages it needs beyond those it holds from the top, until the pages run out: from the first
 * request that needs more than is left on, only those that need none are served.  A request whose pages
 * exceed table_pages, or whose tokens end beyond num_slots, is not served and takes none.
 *
 * Token k of request b is packed row cu_lens[b] + k: positions = cached_lens[b] + k and slots =
 * block_table[b][pos / page_size] * page_size + pos % page_size, or -1 where the request is not served
 * (what the cache producers skip).  seq_lens[b] = cached + new where served, cached where not, 0 where
 * finished.  cu_lens[b] is clamped to num_slots.  Rows from cu_lens[batch] to num_slots: slot -1,
 * position 0.  One or two launches; nothing is allocated.
 */
typedef struct l20_pd_block_tables_args {
  const int32_t *cached_lens;
  const int32_t *new_lens;
  int32_t *block_table;
  int64_t bt_stride_row;
  int32_t table_pages;
  int32_t *free_pages;
  int32_t pool;
  const int32_t *free_count;
  int32_t *free_count_out;
  int64_t *slots;
  int64_t *positions;
  int32_t num_slots;
  int32_t *cu_lens;
  int32_t *seq_lens;
  int32_t batch, page_size;
} l20_pd_block_tables_args;

int32_t l20_pd_block_tables_check(const l20_pd_block_tables_args *args);
int32_t l20_pd_block_tables(const l20_pd_block_tables_args *args, void *stream);

/*
 * Pairs of pages to copy, as the calls below leave them: `src`, `dst` and `tokens` [room] int32 (pages, and
 * how many of the page's first tokens are in use), count [2] int32: how many there are, and how many more
 * were wanted but found no page.  Cells behind the pairs: -1, -1 and 0.
 *
 * l20_pd_reorder_tables: row i of each group of `beams` rows becomes what row parents[i] of the group was (any other
 * value: the row is given up).  A page that several rows hold counts its holders beyond the first in page_shares
 * (0 for every page that one row holds, or none: what l20_pd_block_tables takes needs no entry).
 *
 *   parents     [groups, beams] int32, contiguous
 *   block_table [groups * beams, table_pages] int32, updated: row r holds its first ceil(seq_lens[r] / page_size) cells
 *   seq_lens    [groups * beams] int32, updated: the parent's, 0 where given up
 *   page_shares [pages] int32, updated
 *   free_pages  [pool] int32 stack and free_count [1], updated
 *
 * Full pages are shared.  A last page that is not full is written next, so one child keeps it -- the one in its
 * parent's own row, else the first -- and every other one gets a fresh page and a pair (src, dst, tokens).  Such a
 * page must be held by one row only, which these calls keep true.  Pages that no row holds any more go on top of
 * the stack first, by rising number (what it cannot hold is dropped); then the copies take theirs from the top,
 * row by row.  A row that finds none, or no page number, keeps -1 in that cell and is counted in count[1].  Cells that no row
 * holds are left as they were; numbers outside 0 .. pages - 1 are held by nobody, and children get them as they are, as
 * a last page too.  Pairs: room >= groups * beams.
 * One or two launches.
 */
typedef struct l20_pd_reorder_args {
  const int32_t *parents;
  int32_t *block_table;
  int64_t bt_stride_row;
  int32_t table_pages;
  int32_t *seq_lens;
  int32_t *page_shares;
  int32_t pages;
  int32_t *free_pages;
  int32_t pool;
  int32_t *free_count;
  int32_t *src;
  int32_t *dst;
  int32_t *tokens;
  int32_t room;
  int32_t *count;
  int32_t groups, beams, page_size;
  void *workspace;
  int64_t workspace_bytes;
} l20_pd_reorder_args;

int32_t l20_pd_reorder_tables_check(const l20_pd_reorder_args *args);
/* Bytes of workspace for these groups, beams and table_pages (and for any smaller). */
int64_t l20_pd_reorder_tables_workspace(const l20_pd_reorder_args *args);
int32_t l20_pd_reorder_tables(const l20_pd_reorder_args *args, void *stream);

/*
 * l20_pd_compact_pages: the pool shrinks to the pages below `limit`.  Pages that the table's rows hold at or
 * beyond it move to free pages below it, the lowest to the lowest, as many as there is room for; table, page_shares
 * and stack follow, and the pairs say what to copy (tokens: page_size).  The stack keeps the pages below the limit
 * that are still free, the lowest on top; those beyond it leave the pool.  count[1]: pages that had to stay beyond
 * (the stack gets them back when they are given up).
 * A page that neither the stack nor a row of the table holds stays where it is.
 */
typedef struct l20_pd_compact_args {
  int32_t limit;
  int32_t *block_table;
  int64_t bt_stride_row;
  int32_t table_pages;
  const int32_t *seq_lens;
  int32_t *page_shares;
  int32_t pages;
  int32_t *free_pages;
  int32_t pool;
  int32_t *free_count;
  int32_t *src;
  int32_t *dst;
  int32_t *tokens;
  int32_t room;
  int32_t *count;
  int32_t rows, page_size;
  void *workspace;
  int64_t workspace_bytes;
} l20_pd_compact_args;

int32_t l20_pd_compact_pages_check(const l20_pd_compact_args *args);
/* Bytes of workspace for this number of pages (and for fewer). */
int64_t l20_pd_compact_pages_workspace(const l20_pd_compact_args *args);
int32_t l20_pd_compact_pages(const l20_pd_compact_args *args, void *stream);

/*
 * l20_pd_copy_pages: the first tokens[k] tokens of page src[k] to page dst[k], k < min(*count, room), in each of
 * `num_caches` caches (HOST array of device pointers) of one layout: `pages` pages of stride_page bytes, and in a page
 * up to three levels of (size, stride in bytes), the longest stride first, above `inner` contiguous bytes.
 * token_level: the level that counts tokens (-1: whole pages, `tokens` is not read).  count NULL: all of `room`;
 * tokens NULL: whole pages.  Pairs with a page outside the cache are skipped.  No page may be the dst of two pairs,
 * or dst of one and src of another: such pages hold either.
 */
typedef struct l20_pd_copy_args {
  const int32_t *src;
  const int32_t *dst;
  const int32_t *tokens;
  int32_t room;
  const int32_t *count;
  void *const *caches;
  int32_t num_caches;
  int64_t pages, stride_page;
  int64_t size0, stride0;
  int64_t size1, stride1;
  int64_t size2, stride2;
  int64_t inner;
  int32_t token_level;
} l20_pd_copy_args;

int32_t l20_pd_copy_pages_check(const l20_pd_copy_args *args);
int32_t l20_pd_copy_pages(const l20_pd_copy_args *args, void *stream);

#ifdef __cplusplus
}
#endif

#endif /* L20_BLOCK_TABLES_H_ */
