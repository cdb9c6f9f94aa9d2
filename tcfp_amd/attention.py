"""An 8-bit paged K/V cache and attention over it (HIP, gfx950; no reference
counterpart).

The cache holds, for K and for V, E4M3 codes ``[pages, kv_heads, page_size,
dim]`` and one power-of-two exponent per token and head (int8 ``[pages,
kv_heads, page_size]``): the block format of ``kernels.block_quantize_fp8``
with the head as the block.  A token's place is its *slot*, ``page * page_size
+ place in the page``; which pages a sequence has is its row of a page table.

* :func:`kv_cache_write` quantises new keys and values into their slots,
* :func:`kv_cache_read` reads slots back,
* :func:`paged_attention` attends new tokens -- one per sequence when
  generating, thousands for a prompt or a part of one -- over the cache,
* :class:`PagedKVCache` owns a pool of pages for every layer of a model and
  hands them out to sequences.

The lengths of a batch are read on the device, so a captured graph can be
replayed as they grow.  Every op runs on the tensors' GPU and current stream;
there is no CPU path.
"""
from __future__ import annotations

import torch

from . import _hip

__all__ = ["kv_cache_write", "kv_cache_read", "paged_attention"]


def kv_cache_write(
    k: torch.Tensor,
    v: torch.Tensor,
    k_codes: torch.Tensor,
    v_codes: torch.Tensor,
    k_exps: torch.Tensor,
    v_exps: torch.Tensor,
    slots: torch.Tensor,
) -> None:
    """Quantise ``k`` and ``v`` [tokens, kv_heads, dim] (fp32 or bf16; slices
    of a QKV projection's output are taken as they are) into the cache's
    ``slots`` (int64 [tokens], all different).

    A slot below 0 or past the pool leaves its token out (the padding of a
    batch of fixed size).  Values that are not finite become NaN codes and
    leave the exponent of the others alone.
    """
    _hip.host().kv_cache_write(k, v, k_codes, v_codes, k_exps, v_exps, slots)


def kv_cache_read(
    k_codes: torch.Tensor,
    v_codes: torch.Tensor,
    k_exps: torch.Tensor,
    v_exps: torch.Tensor,
    slots: torch.Tensor,
    *,
    out_dtype: torch.dtype = torch.bfloat16,
) -> tuple[torch.Tensor, torch.Tensor]:
    """``(k, v)`` [tokens, kv_heads, dim] of the cache's ``slots`` (int64), in
    fp32 or bf16 (both hold a cached value exactly); zeros where a slot is
    outside the pool."""
    return _hip.host().kv_cache_read(k_codes, v_codes, k_exps, v_exps, slots, out_dtype)


def paged_attention(
    q: torch.Tensor,
    k_codes: torch.Tensor,
    v_codes: torch.Tensor,
    k_exps: torch.Tensor,
    v_exps: torch.Tensor,
    page_table: torch.Tensor,
    seq_lens: torch.Tensor,
    query_start: torch.Tensor,
    *,
    max_query_len: int,
    max_seq_len: int | None = None,
    scale: float | None = None,
    causal: bool = True,
    window: int = 0,
) -> torch.Tensor:
    """Attention of a batch's new tokens over the paged cache, bf16 [tokens,
    heads, dim].

    ``q`` [tokens, heads, dim] bf16 holds the new tokens of all sequences one
    after another, sequence b's in rows ``query_start[b]`` to
    ``query_start[b + 1]`` (int32 [sequences + 1]); ``seq_lens`` (int32) is
    each sequence's number of cached tokens, the new ones -- already written
    -- last; ``page_table`` (int32 [sequences, pages]) its pages in order.
    ``heads`` is a multiple of the cache's heads, neighbouring query heads
    share one.

    A token at position p of its sequence sees the keys up to p (``causal``)
    that are less than ``window`` positions back (``window`` > 0); without
    ``causal`` it sees all keys of the sequence, within the window behind it.
    Keys on a page outside the pool (-1: given up because no window reaches
    it) are not seen; a token that sees nothing, and one that belongs to no
    sequence, gets zeros.  ``scale`` is ``dim ** -0.5`` by default.

    ``max_query_len`` and ``max_seq_len`` (by default what the table spans)
    bound the batch's lengths and size the launch.
    """
    return _hip.host().paged_attention(q, k_codes, v_codes, k_exps, v_exps, page_table, seq_lens,
                                       query_start, int(max_query_len),
                                       None if max_seq_len is None else int(max_seq_len),
                                       None if scale is None else float(scale), bool(causal),
                                       int(window))
