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

from dataclasses import dataclass

import torch

from . import _hip

__all__ = ["kv_cache_write", "kv_cache_read", "paged_attention", "PagedKVCache", "CacheBatch"]


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
    fp32 or bf16 (both hold a cached value exactly, bf16 but for values under
    its smallest); zeros where a slot is outside the pool."""
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
    sequence, gets zeros.  A NaN in a cached key reaches the tokens that see it,
    one in a cached value its own column of them, and neither anything else.
    ``scale`` is ``dim ** -0.5`` by default.

    ``max_query_len`` and ``max_seq_len`` (by default what the table spans)
    bound the batch's lengths and size the launch.

    For serving: there is no backward pass.  Where ``q`` requires a gradient the
    result does too, and a backward pass that reaches it raises
    ``NotImplementedError``.
    """
    out = _hip.host().paged_attention(q, k_codes, v_codes, k_exps, v_exps, page_table, seq_lens,
                                      query_start, int(max_query_len),
                                      None if max_seq_len is None else int(max_seq_len),
                                      None if scale is None else float(scale), bool(causal),
                                      int(window))
    if torch.is_grad_enabled() and q.requires_grad:
        return _NoBackward.apply(q, out)
    return out


class _NoBackward(torch.autograd.Function):
    """Ties ``paged_attention``'s result to its ``q``, so that a gradient is not
    lost without a word."""

    @staticmethod
    def forward(ctx, q, out):
        return out.view_as(out)

    @staticmethod
    def backward(ctx, grad):
        raise NotImplementedError("paged_attention has no backward pass (the cache holds "
                                  "quantised keys and values, for serving)")


@dataclass
class CacheBatch:
    """One step of a batch of sequences: where its new tokens go and what they
    see (the index arguments of :func:`kv_cache_write` and
    :func:`paged_attention`), the same for every layer of a model."""

    slots: torch.Tensor        # int64 [new tokens]
    page_table: torch.Tensor   # int32 [sequences, pages]
    seq_lens: torch.Tensor     # int32 [sequences], the new tokens counted
    query_start: torch.Tensor  # int32 [sequences + 1]
    max_query_len: int
    max_seq_len: int


class PagedKVCache:
    """A pool of pages for the keys and values of every layer of a model, and
    the page lists of the sequences that live in it.

    ``open()`` starts a sequence, ``extend()`` makes room for its new tokens
    (and describes the step to the ops), ``close()`` gives its pages back.
    A page holds ``page_size`` tokens of one sequence, in every layer.
    """

    def __init__(self, layers: int, pages: int, kv_heads: int, dim: int, *, page_size: int = 64,
                 device: torch.device | str = "cuda") -> None:
        if layers < 1 or pages < 1 or kv_heads < 1:
            raise ValueError("a cache needs at least one layer, page and head")
        if dim not in (64, 128, 256):
            raise ValueError(f"the head dimension must be 64, 128 or 256, got {dim}")
        if page_size < 16 or page_size > 1024 or page_size & (page_size - 1):
            raise ValueError(f"page_size must be a power of two from 16 to 1024, got {page_size}")
        self.page_size, self.device = page_size, torch.device(device)
        shape = (layers, pages, kv_heads, page_size)
        self.k_codes, self.v_codes = (
            torch.zeros((*shape, dim), dtype=torch.uint8, device=device).view(torch.float8_e4m3fn)
            for _ in range(2))
        self.k_exps, self.v_exps = (torch.zeros(shape, dtype=torch.int8, device=device)
                                    for _ in range(2))
        self._free = list(range(pages - 1, -1, -1))
        self._pages: dict[int, list[int]] = {}
        self._len: dict[int, int] = {}
        self._next = 0

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def length(self, seq: int) -> int:
        """Tokens of a sequence."""
        return self._len[seq]

    def open(self) -> int:
        """A new, empty sequence."""
        seq = self._next
        self._next += 1
        self._pages[seq], self._len[seq] = [], 0
        return seq

    def close(self, seq: int) -> None:
        """Give a sequence's pages back."""
        self._free.extend(reversed(self._pages.pop(seq)))
        del self._len[seq]

    def extend(self, seqs: list[int], counts: list[int]) -> CacheBatch:
        """Room for ``counts[i]`` new tokens of sequence ``seqs[i]``; the step
        of a batch in that order.  Raises ``RuntimeError`` and changes nothing
        when the pool has too few free pages."""
        if len(seqs) != len(counts) or len(set(seqs)) != len(seqs) or min(counts, default=0) < 0:
            raise ValueError("one count of at least 0 for each of a list of different sequences")
        page = self.page_size
        need = [-(-(self._len[s] + n) // page) - len(self._pages[s]) for s, n in zip(seqs, counts)]
        if sum(need) > len(self._free):
            raise RuntimeError(
                f"the cache has {len(self._free)} free pages, the step needs {sum(need)}")
        slots, lens, starts = [], [], [0]
        for s, n, more in zip(seqs, counts, need):
            mine = self._pages[s]
            mine.extend(self._free.pop() for _ in range(more))
            at = self._len[s]
            slots.extend(mine[j // page] * page + j % page for j in range(at, at + n))
            self._len[s] = at + n
            lens.append(at + n)
            starts.append(starts[-1] + n)
        width = max([len(self._pages[s]) for s in seqs] + [1])
        table = [self._pages[s] + [-1] * (width - len(self._pages[s])) for s in seqs]

        def tensor(v, dtype):
            return torch.tensor(v, dtype=dtype).to(self.device)

        return CacheBatch(
            tensor(slots, torch.int64), tensor(table, torch.int32).reshape(len(seqs), width),
            tensor(lens, torch.int32), tensor(starts, torch.int32), max(counts, default=0),
            max(lens, default=0))

    def layer(self, i: int) -> tuple[torch.Tensor, ...]:
        """``(k_codes, v_codes, k_exps, v_exps)`` of a layer, as the ops take
        them."""
        return self.k_codes[i], self.v_codes[i], self.k_exps[i], self.v_exps[i]

    def write(self, layer: int, k: torch.Tensor, v: torch.Tensor, batch: CacheBatch) -> None:
        """:func:`kv_cache_write` of a step's new tokens."""
        kv_cache_write(k, v, *self.layer(layer), batch.slots)

    def read(self, layer: int, seq: int, *, out_dtype: torch.dtype = torch.bfloat16):
        """:func:`kv_cache_read` of a whole sequence: ``(k, v)`` [tokens,
        kv_heads, dim]."""
        page, pages = self.page_size, self._pages[seq]
        slots = torch.tensor([pages[j // page] * page + j % page for j in range(self._len[seq])],
                             dtype=torch.int64).to(self.device)
        return kv_cache_read(*self.layer(layer), slots, out_dtype=out_dtype)

    def attend(self, layer: int, q: torch.Tensor, batch: CacheBatch, **kw) -> torch.Tensor:
        """:func:`paged_attention` of a step's new tokens (their keys and
        values written)."""
        return paged_attention(q, *self.layer(layer), batch.page_table, batch.seq_lens,
                               batch.query_start, max_query_len=batch.max_query_len,
                               max_seq_len=batch.max_seq_len, **kw)
