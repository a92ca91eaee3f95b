"""Block tables, slot maps and positions of a batch, and its page pool, on the GPU (MI355X).

Every paged operator here takes a block table, lengths and (the cache producers) positions and a slot map.
``l20_build_block_tables`` makes them in one or two launches from the lengths alone, with the page pool as a
stack in device memory: no host round trip in a serving step.

Requests of several hypotheses (beams, parallel samples) are groups of rows.  ``l20_reorder_block_tables`` lets the
rows of a group follow their parents: full pages are shared, a last page in use is copied on write, and pages that
no row holds go back to the pool.  ``l20_compact_pages`` shrinks the pool, and ``l20_copy_pages`` copies what both ask
for, in the caches of all layers.  The reference's callers do this on the host, so these names have no counterpart
there.
"""

from __future__ import annotations

from functools import lru_cache
from typing import NamedTuple, Optional, Sequence

import torch

import l20_paged_decode  # noqa: F401  (loads the ops library)
from l20_paged_split_kv import _gpu_facts

MAX_REQUESTS = 8192


def _need_gpu(name: str, tensor: torch.Tensor) -> None:
    if not (tensor.is_cuda and _gpu_facts(tensor.device)[0]):
        raise RuntimeError(f"{name} requires an MI355X (gfx950) GPU")


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
    _need_gpu("l20_build_block_tables", block_table)
    if cached_lens.ndim != 1 or not 0 <= cached_lens.shape[0] <= MAX_REQUESTS:
        raise RuntimeError(f"cached_lens must be [requests] with at most {MAX_REQUESTS} requests")
    torch.ops.l20_stack.build_block_tables(cached_lens, new_lens, block_table, free_pages, free_count, slot_mapping,
                                           positions, cu_seqlens, seq_lens, int(page_size),
                                           free_count if free_count_out is None else free_count_out)


class PageCopies(NamedTuple):
    """Pairs of pages for ``l20_copy_pages``: ``src``, ``dst`` and ``tokens`` int32 [room] (how many of the page's first
    tokens are in use), ``count`` int32 [2]: the pairs, and how many more were wanted but found no page.  Without
    ``tokens`` whole pages are copied, without ``count`` all of them."""

    src: torch.Tensor
    dst: torch.Tensor
    tokens: Optional[torch.Tensor] = None
    count: Optional[torch.Tensor] = None

    @staticmethod
    def empty(room: int, device) -> "PageCopies":
        return PageCopies(*(torch.empty(n, dtype=torch.int32, device=device) for n in (room, room, room, 2)))


@lru_cache(maxsize=4096)
def _workspace_bytes(kind: str, **sizes: int) -> int:
    import l20_pd_cabi

    a = {"reorder_tables": l20_pd_cabi.L20PdReorderArgs, "compact_pages": l20_pd_cabi.L20PdCompactArgs}[kind](**sizes)
    return int(getattr(l20_pd_cabi.load(), f"l20_pd_{kind}_workspace")(l20_pd_cabi.ctypes.byref(a)))


def allocate_l20_reorder_workspace(parents: torch.Tensor, block_table: torch.Tensor) -> torch.Tensor:
    """The workspace of ``l20_reorder_block_tables`` for up to these groups and this width of the table (int32).  Calls
    that may overlap each need their own; its contents do not matter."""
    size = _workspace_bytes("reorder_tables", groups=parents.shape[0], beams=parents.shape[1],
                            table_pages=block_table.shape[1])
    return torch.empty(size // 4, dtype=torch.int32, device=block_table.device)


def l20_reorder_block_tables(
    parents: torch.Tensor,
    block_table: torch.Tensor,
    seq_lens: torch.Tensor,
    page_shares: torch.Tensor,
    free_pages: torch.Tensor,
    free_count: torch.Tensor,
    page_size: int,
    *,
    copies: Optional[PageCopies] = None,
    workspace: Optional[torch.Tensor] = None,
) -> PageCopies:
    """Row i of each group becomes what row ``parents[group, i]`` of the group was; -1: the row is given up.

    ``parents`` int32 [groups, beams] as ``l20_beam_search_step`` gives them; ``block_table`` [groups * beams, pages]
    and ``seq_lens`` [groups * beams] (int32, updated in place): row r holds the first ``ceil(seq_lens[r] / page_size)``
    cells.  ``page_shares`` int32 [pages] counts the rows beyond the first that hold a page and is 0 to begin with;
    ``free_pages`` and ``free_count`` are the pool of ``l20_build_block_tables``, whose pages need no entry.

    Full pages are shared.  A last page that is not full stays with one child (the one in its parent's own row, else
    the first); every other child gets a fresh page, and a pair that says which tokens to copy to it.  Pages that no
    row holds any more go on top of the stack by rising number, before fresh ones are taken.  A group of one length takes as
    many pages more than it gives back as it has live rows more than before: to be sure of them the stack has to hold
    ``beams`` less its live rows for every group, also those that a step gave back which left fewer.  A row that finds none
    keeps -1 in that cell and is counted in ``count[1]``: its tokens there, and its children's, are masked by the attention
    and skipped by the producers.

    Rows that share pages are given up here, and not by ``l20_build_block_tables``, which knows no shares; a page that
    is not full must be held by one row, which both keep true.  With ``copies`` (room for a pair a row) and
    ``workspace`` given nothing is allocated and the call can be captured in a graph."""
    _need_gpu("l20_reorder_block_tables", block_table)
    if parents.ndim != 2:
        raise RuntimeError("parents must be [groups, beams]")
    if copies is None:
        copies = PageCopies.empty(parents.numel(), block_table.device)
    if workspace is None:
        workspace = allocate_l20_reorder_workspace(parents, block_table)
    torch.ops.l20_stack.reorder_block_tables(parents, block_table, seq_lens, page_shares, free_pages, free_count,
                                             int(page_size), *copies, workspace)
    return copies


def allocate_l20_compact_workspace(page_shares: torch.Tensor) -> torch.Tensor:
    """The workspace of ``l20_compact_pages`` for up to these pages (int32); its contents do not matter."""
    return torch.empty(_workspace_bytes("compact_pages", pages=page_shares.shape[0]) // 4, dtype=torch.int32,
                       device=page_shares.device)


def l20_compact_pages(
    limit: int,
    block_table: torch.Tensor,
    seq_lens: torch.Tensor,
    page_shares: torch.Tensor,
    free_pages: torch.Tensor,
    free_count: torch.Tensor,
    page_size: int,
    *,
    copies: Optional[PageCopies] = None,
    workspace: Optional[torch.Tensor] = None,
) -> PageCopies:
    """Shrink the pool to the pages below ``limit``: what the table's rows hold at or beyond it moves to free pages below.

    The lowest such page moves to the lowest free one, and so on, as long as there is room (in ``copies`` too: by default
    for every cell of the table or page of the pool, whichever are fewer); ``count[1]`` says how many had to stay.
    ``block_table``, ``page_shares`` and the stack follow: it keeps the pages below ``limit`` that are still free, the
    lowest on top, and those beyond leave the pool.  The contents are still to be copied (``l20_copy_pages``, whole
    pages).  A page that neither the stack nor a row of the table holds stays where it is, so every table that shares
    pages with this one has to be in the call."""
    _need_gpu("l20_compact_pages", block_table)
    if copies is None:
        copies = PageCopies.empty(min(block_table.numel(), page_shares.numel()), block_table.device)
    if workspace is None:
        workspace = allocate_l20_compact_workspace(page_shares)
    torch.ops.l20_stack.compact_pages(int(limit), block_table, seq_lens, page_shares, free_pages, free_count,
                                      int(page_size), *copies, workspace)
    return copies


def l20_copy_pages(copies: PageCopies, caches: Sequence[torch.Tensor]) -> None:
    """Copy the pairs of pages in every one of ``caches``: tensors [pages, page, ...] of any type and of any order of
    dimensions inside a page (key and value caches of all layers, latent caches); those of one layout go in one launch.

    Only the first ``tokens`` tokens of a page are copied; what lies behind them is left as it was.  Pairs with a page
    outside a cache are skipped.  No page may be the ``dst`` of two pairs, or of one and ``src`` of another."""
    _need_gpu("l20_copy_pages", copies.src)
    torch.ops.l20_stack.copy_pages(*copies, caches)


def _register_fake() -> None:
    @torch.library.register_fake("l20_stack::build_block_tables")
    def _build_block_tables_fake(cached_lens, new_lens, block_table, free_pages, free_count, slot_mapping, positions,
                                 cu_seqlens, seq_lens, page_size, free_count_out):
        return None

    @torch.library.register_fake("l20_stack::reorder_block_tables")
    def _reorder_block_tables_fake(parents, block_table, seq_lens, page_shares, free_pages, free_count, page_size, src,
                                   dst, tokens, count, workspace):
        return None

    @torch.library.register_fake("l20_stack::compact_pages")
    def _compact_pages_fake(limit, block_table, seq_lens, page_shares, free_pages, free_count, page_size, src, dst,
                            tokens, count, workspace):
        return None

    @torch.library.register_fake("l20_stack::copy_pages")
    def _copy_pages_fake(src, dst, tokens, count, caches):
        return None


_register_fake()
