"""Block tables, slot maps and positions of a batch from its request lengths, on the GPU (MI355X).

Every paged operator here takes a block table, lengths and (the cache producers) positions and a slot map.
``l20_build_block_tables`` makes them in one or two launches from the lengths alone, with the page pool as a
stack in device memory: no host round trip in a serving step.  The reference's callers build them on the host,
so this name has no counterpart there.
"""

from __future__ import annotations

from typing import Optional

import torch

import l20_paged_decode  # noqa: F401  (loads the ops library)
from l20_paged_split_kv import _gpu_facts

MAX_REQUESTS = 8192


def l20_build_block_tables(
    cached_lens: torch.Tensor,
    new_lens: torch.Tensor,
    block_table: torch.Tensor,
    free_pages: torch.Tensor,
    free_count: torch.Tensor,
    slot_mapping: torch.Tensor,
    positions: torch.Tensor,
    cu_seqlens: torch.Tensor,
    seq_lens: torch.Tensor,
    page_size: int,
    *,
    free_count_out: Optional[torch.Tensor] = None,
) -> None:
    """Append ``new_lens[b]`` tokens to requests of ``cached_lens[b]`` tokens (below 0: the request is finished).

    ``block_table`` [requests, pages] and the stack ``free_pages`` [pool] with its ``free_count`` [1] are int32 and
    updated in place (``free_count_out``: another tensor for the new count).  First the pages of finished requests
    go on top of the stack; then the requests are served in order, each taking the pages it lacks from the top,
    until they run out.  A request that finds too few, or exceeds its table row, or whose tokens end beyond
    ``slot_mapping``, is not served: its slots are -1 (the cache producers skip them) and ``seq_lens[b]`` stays
    ``cached_lens[b]``.  Once one finds too few pages, later ones are served only if they need none.

    Outputs: ``slot_mapping`` and ``positions`` int64 [tokens] in packed order (rows past the last token: slot -1,
    position 0), ``cu_seqlens`` int32 [requests + 1], ``seq_lens`` int32 [requests] (0 where finished; not the same
    tensor as ``cached_lens``)."""
    if not (block_table.is_cuda and _gpu_facts(block_table.device)[0]):
        raise RuntimeError("l20_build_block_tables requires an MI355X (gfx950) GPU")
    if cached_lens.ndim != 1 or not 0 <= cached_lens.shape[0] <= MAX_REQUESTS:
        raise RuntimeError(f"cached_lens must be [requests] with at most {MAX_REQUESTS} requests")
    torch.ops.l20_stack.build_block_tables(cached_lens, new_lens, block_table, free_pages, free_count, slot_mapping,
                                           positions, cu_seqlens, seq_lens, int(page_size),
                                           free_count if free_count_out is None else free_count_out)


def _register_fake() -> None:
    @torch.library.register_fake("l20_stack::build_block_tables")
    def _build_block_tables_fake(cached_lens, new_lens, block_table, free_pages, free_count, slot_mapping, positions,
                                 cu_seqlens, seq_lens, page_size, free_count_out):
        return None


_register_fake()
