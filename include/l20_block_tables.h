/*
 * C ABI of the block-table builder in libl20_paged_decode_hip.so: a batch's block tables, slot map,
 * positions and lengths from its request lengths, on the GPU.  Return codes and l20_pd_last_error() are
 * those of l20_paged_decode.h.  The reference's callers build these on the host: no counterpart there.
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

#ifdef __cplusplus
}
#endif

#endif /* L20_BLOCK_TABLES_H_ */
