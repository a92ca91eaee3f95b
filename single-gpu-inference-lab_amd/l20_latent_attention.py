"""Latent attention for MI355X: one latent vector a token is key and value of every head.

A model with latent attention projects each token down to ``rank`` latent values and a rotary key part of
64 dims, and keeps only those: ``latent_cache`` is ``[pages, page, rank + 64]``, in the model's type or
``float8_e4m3fn`` (with one ``cache_scale``).  Three functions, in the order of a serving step:

* ``l20_latent_rope_and_cache`` -- norm of the latent, RoPE of key and query parts, the paged cache write;
* ``l20_latent_prompt_attention`` -- causal attention of prompts, over keys and values expanded from the
  latents by the model's up-projection (expanded form);
* ``l20_paged_latent_attention`` -- decode and verification steps over the paged cache, with the key
  up-projection absorbed into the query and the value up-projection applied to the output (absorbed form).

Block tables, slot maps and positions come from ``l20_block_tables``.  All call ``torch.ops.l20_stack`` ops of
the native library on the current stream; there is no CPU fallback, and no backward pass: the framework serves.
The reference has no latent attention, so these names have no counterpart there.
"""

from __future__ import annotations

from functools import lru_cache
from typing import Optional

import torch

import l20_paged_decode  # noqa: F401  (loads the ops library)
from l20_paged_split_kv import _gpu_facts, gpu_cus

ROPE_DIM = 64
RANKS = (256, 512)
HEAD_DIM = 128  # key and value dims of a head in the expanded form


def _need_gpu(name: str, tensor: torch.Tensor) -> None:
    if not (tensor.is_cuda and _gpu_facts(tensor.device)[0]):
        raise RuntimeError(f"{name} requires an MI355X (gfx950) GPU")


def _cache_ok(cache: torch.Tensor, dtype: torch.dtype, rank: int) -> None:
    if cache.ndim != 3 or cache.shape[2] != rank + ROPE_DIM or rank not in RANKS:
        raise RuntimeError("latent cache must be [pages, page, rank + 64] with rank 256 or 512")
    if cache.dtype not in (torch.float8_e4m3fn, dtype):
        raise RuntimeError("latent cache must be torch.float8_e4m3fn or the model dtype")


# (sizes from shapes alone; the calls into the library take longer than a small kernel)
@lru_cache(maxsize=4096)
def _paged_bytes(batch: int, q_len: int, heads: int, rank: int, max_seq_len: int, cache_dtype: torch.dtype, cus: int) -> int:
    import l20_pd_cabi

    a = l20_pd_cabi.L20PdLatentArgs()
    a.batch, a.q_len, a.num_heads, a.rank, a.max_seq_len = batch, q_len, heads, rank, max_seq_len
    a.cache_dtype = l20_pd_cabi._kv_code(torch.empty(0, dtype=cache_dtype))
    return int(l20_pd_cabi.load().l20_pd_paged_latent_workspace(l20_pd_cabi.ctypes.byref(a), cus))


@lru_cache(maxsize=4096)
def _prompt_bytes(total_q: int, heads: int, total_k: int, batch: int, max_q: int, cus: int) -> int:
    import l20_pd_cabi

    a = l20_pd_cabi.L20PdLatentPromptArgs()
    a.total_q, a.num_heads, a.total_k, a.batch, a.max_q_len = total_q, heads, total_k, batch, max_q
    return int(l20_pd_cabi.load().l20_pd_latent_prompt_workspace(l20_pd_cabi.ctypes.byref(a), cus))


def l20_latent_rope_and_cache(
    query_rope: Optional[torch.Tensor],
    latent: torch.Tensor,
    key_rope: torch.Tensor,
    positions: torch.Tensor,
    cos_sin_cache: torch.Tensor,
    is_neox: bool,
    latent_cache: torch.Tensor,
    slot_mapping: torch.Tensor,
    *,
    norm_weight: Optional[torch.Tensor] = None,
    norm_eps: float = 1e-6,
    cache_scale: float = 1.0,
    query_out: Optional[torch.Tensor] = None,
    latent_out: Optional[torch.Tensor] = None,
    key_rope_out: Optional[torch.Tensor] = None,
) -> None:
    """Norm (with ``norm_weight``) and RoPE of new tokens, and their rows into the paged cache.

    ``query_rope`` [tokens, heads, 64] (or None), ``latent`` [tokens, rank] and ``key_rope`` [tokens, 64] are views
    of any row stride; each result goes to its ``_out`` tensor, or in place where none is given (an ``_out`` tensor that
    is not its input must share no bytes with the inputs). A ``query_out``
    that is the last 64 dims of the absorbed query saves the copy there. ``slot_mapping`` below 0 or beyond the
    cache: the token is not stored; two tokens of a call must not name one slot. An fp8 cache stores ``clamp(x /
    cache_scale)`` of the rounded results."""
    _need_gpu("l20_latent_rope_and_cache", latent)
    # (shapes and strides are checked by the op: a second time here they would take as long as the kernel)
    if latent.dtype not in (torch.float16, torch.bfloat16):
        raise RuntimeError("l20_latent_rope_and_cache supports FP16 and BF16")
    if query_rope is None and query_out is not None:
        raise RuntimeError("query_out needs query_rope")
    torch.ops.l20_stack.latent_rope_and_cache(
        query_rope, latent, key_rope, positions, cos_sin_cache, bool(is_neox), latent_cache, slot_mapping,
        query_rope if query_out is None else query_out, latent if latent_out is None else latent_out,
        key_rope if key_rope_out is None else key_rope_out, norm_weight, float(norm_eps), float(cache_scale))


def allocate_l20_paged_latent_workspace(
    query: torch.Tensor,
    latent_cache: torch.Tensor,
    max_seq_len: int,
    *,
    kv_rank: int = 512,
    q_len: int = 1,
) -> torch.Tensor:
    """The workspace of ``l20_paged_latent_attention`` for queries of up to this many sequences (and these heads and
    ``q_len``) and bounds up to ``max_seq_len`` (uint8; empty where none is needed).  Calls that may overlap each need
    their own; its contents do not matter."""
    size = _paged_bytes(query.shape[0] // q_len, q_len, query.shape[1], kv_rank, int(max_seq_len), latent_cache.dtype,
                        gpu_cus(latent_cache.device))
    return torch.empty(size, dtype=torch.uint8, device=latent_cache.device)


def l20_paged_latent_attention(
    query: torch.Tensor,
    latent_cache: torch.Tensor,
    block_table: torch.Tensor,
    seq_lens: torch.Tensor,
    *,
    softmax_scale: float,
    kv_rank: int = 512,
    cache_scale: float = 1.0,
    max_seq_len: Optional[int] = None,
    q_len: int = 1,
    output: Optional[torch.Tensor] = None,
    workspace: Optional[torch.Tensor] = None,
    lse: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """Attention of ``query`` [batch * q_len, heads, kv_rank + 64] over a paged latent cache; returns ``output``
    [batch * q_len, heads, kv_rank], to which the model applies its value up-projection.

    Row b * q_len + i sees the first ``seq_lens[b] - q_len + i + 1`` tokens of sequence b; one that sees none gives
    zeros (``lse``: -inf). ``output`` must not share bytes with ``query``. ``softmax_scale`` is the model's (its head dims
    before the absorption, not ``kv_rank``, set it). ``max_seq_len`` bounds the lengths (default: what the block
    table can name) and sizes grid and workspace; tokens beyond it, the table, or on a page outside the cache are
    masked. With ``output`` and ``workspace`` given nothing is allocated and the call can be captured in a graph."""
    _need_gpu("l20_paged_latent_attention", query)
    if query.ndim != 3 or query.dtype not in (torch.float16, torch.bfloat16):
        raise RuntimeError("expected an FP16 or BF16 query [batch * q_len, heads, kv_rank + 64]")
    _cache_ok(latent_cache, query.dtype, kv_rank)
    if query.shape[2] != kv_rank + ROPE_DIM or q_len < 1 or query.shape[0] % q_len:
        raise RuntimeError("expected query [batch * q_len, heads, kv_rank + 64]")
    if block_table.ndim != 2:
        raise RuntimeError("block table must be int32 [batch, pages] with contiguous rows")
    if max_seq_len is None:
        max_seq_len = block_table.shape[1] * latent_cache.shape[1]
    if output is None:
        output = query.new_empty(*query.shape[:2], kv_rank)
    elif output.shape != (*query.shape[:2], kv_rank):
        raise RuntimeError("output must be [batch * q_len, heads, kv_rank]")
    if workspace is None:
        workspace = allocate_l20_paged_latent_workspace(query, latent_cache, max_seq_len, kv_rank=kv_rank, q_len=q_len)
    return torch.ops.l20_stack.paged_latent_attention_out(query, latent_cache, block_table, seq_lens, output, workspace,
                                                          float(softmax_scale), float(cache_scale), int(max_seq_len),
                                                          int(q_len), lse)


def allocate_l20_latent_prompt_workspace(
    query: torch.Tensor,
    key: torch.Tensor,
    batch: int,
    max_seqlen_q: int,
) -> torch.Tensor:
    """The workspace of ``l20_latent_prompt_attention`` for exactly these shapes (uint8; empty where the keys are not
    split: the call then takes an empty one, and does not split).  Calls that may overlap each need their own; its
    contents do not matter."""
    size = _prompt_bytes(query.shape[0], query.shape[1], key.shape[0], batch, int(max_seqlen_q), gpu_cus(query.device))
    return torch.empty(size, dtype=torch.uint8, device=query.device)


def l20_latent_prompt_attention(
    query: torch.Tensor,
    key: torch.Tensor,
    key_rope: torch.Tensor,
    value: torch.Tensor,
    cu_seqlens_q: torch.Tensor,
    cu_seqlens_k: torch.Tensor,
    max_seqlen_q: int,
    *,
    softmax_scale: Optional[float] = None,
    causal: bool = True,
    output: Optional[torch.Tensor] = None,
    workspace: Optional[torch.Tensor] = None,
    lse: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """Attention of packed prompts: ``query`` [tokens, heads, 192] (its last 64 dims rotated), ``key`` and
    ``value`` [key tokens, heads, 128] (views of the up-projection's output, say), ``key_rope`` [key tokens, 64]
    shared by the heads; returns ``output`` [tokens, heads, 128].

    Sequence b has the query rows and the keys of its ``cu_seqlens`` ranges; with ``causal`` query i of n sees
    keys up to i + (keys - n), so that a chunk whose first tokens are cached already passes all keys.  A row that
    sees none gives zeros (``lse``: -inf); rows outside the ranges, or beyond ``max_seqlen_q``, keep what they
    held.  ``output`` must not share bytes with an input.  ``softmax_scale`` defaults to 192^-0.5.  Calls of few rows and many keys split the keys, with a
    ``workspace`` (default: allocated)."""
    _need_gpu("l20_latent_prompt_attention", query)
    if query.dtype not in (torch.float16, torch.bfloat16):
        raise RuntimeError("l20_latent_prompt_attention supports FP16 and BF16")
    if query.ndim != 3 or query.shape[2] != HEAD_DIM + ROPE_DIM:
        raise RuntimeError("expected query [tokens, heads, 192]")
    if key.ndim != 3 or value.shape != key.shape or key.shape[1:] != (query.shape[1], HEAD_DIM):
        raise RuntimeError("expected key and value [key tokens, heads, 128]")
    if output is None:
        output = query.new_empty(*query.shape[:2], HEAD_DIM)
    if softmax_scale is None:
        softmax_scale = (HEAD_DIM + ROPE_DIM) ** -0.5
    if workspace is None and cu_seqlens_q.ndim == 1 and cu_seqlens_q.shape[0] > 1:
        size = _prompt_bytes(query.shape[0], query.shape[1], key.shape[0], cu_seqlens_q.shape[0] - 1, int(max_seqlen_q),
                             gpu_cus(query.device))
        workspace = torch.empty(size, dtype=torch.uint8, device=query.device) if size else None
    return torch.ops.l20_stack.latent_prompt_attention_out(query, key, key_rope, value, cu_seqlens_q, cu_seqlens_k,
                                                           int(max_seqlen_q), output, float(softmax_scale), bool(causal),
                                                           lse, workspace)


def _register_fake() -> None:
    @torch.library.register_fake("l20_stack::latent_rope_and_cache")
    def _latent_rope_and_cache_fake(query, latent, key_rope, positions, cos_sin_cache, is_neox, latent_cache,
                                    slot_mapping, query_out, latent_out, key_rope_out, norm_weight=None, norm_eps=1e-6,
                                    cache_scale=1.0):
        return None

    @torch.library.register_fake("l20_stack::paged_latent_attention_out")
    def _paged_latent_attention_fake(query, latent_cache, block_table, seq_lens, output, workspace, softmax_scale,
                                     cache_scale, max_seq_len, q_len=1, lse=None):
        return output

    @torch.library.register_fake("l20_stack::latent_prompt_attention_out")
    def _latent_prompt_attention_fake(query, key, key_rope, value, cu_seqlens_q, cu_seqlens_k, max_seqlen_q, output,
                                      softmax_scale, causal=True, lse=None, workspace=None):
        return output


_register_fake()
