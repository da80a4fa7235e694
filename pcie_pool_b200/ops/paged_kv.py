"""Operators on the paged KV cache of one layer: attention of one new token per
request, the key bounds of the cache's pages, the blocks that sparse attention
reads, and the blocks that may leave the GPU.

The cache of a layer is ``[2, pages, block, kv_heads, dim]``, K then V, in any
strides that are multiples of 16 bytes with a contiguous last dimension; a
``[pages, 2, ...]`` cache is passed as ``kv.transpose(0, 1)`` (to these operators
only: the offloaders take it as it is).  Request ``b`` holds ``context_lens[b]`` tokens, block
``j`` of it in page ``block_table[b, j]``.  A table entry that is no page
(negative, or ``>= pages``) is a block that is not resident -- offloaded, say --
and its tokens are left out.  Where a batch's table is as wide as the longest
request may get, pass the columns that its requests use (``table[:, :n]``): block
mass, selection and eviction go by the width (256 requests of 100 tokens with
mass take 34 us with 7 columns and 239 with 8192).  Lengths and tables are read on the device when the
kernel runs, so all calls can be captured into a CUDA graph and replayed with
other contents.

A serving step with a bounded cache strings them together::

    out = paged_kv_attention(q, kv, table, lens, mass=mass)          # every layer adds to mass
    e = paged_kv_evict(mass, table, lens, budget, block_size=16)     # pages e.evicted_blocks leave
    # PagedKVOffloader.save(...) them, then go on with e.block_table, e.context_lens, e.mass
    # (PagedKVOffloader.evict(...) does both, and says which of the pages nobody holds any more)

and one with sparse reads::

    paged_kv_bounds(kv, table, lens, bounds, new_tokens=1)
    blocks = paged_kv_select(q, bounds, table, lens, keep, block_size=16)
    out = paged_kv_attention(q, kv, table, lens, blocks=blocks)

All run on the tensors' device and its current stream, without a synchronisation,
and raise ``ValueError`` for what they do not take; none has a gradient.
"""

from __future__ import annotations

from typing import NamedTuple

from .._native import native_kv


def paged_kv_attention(q, kv, block_table, context_lens, *, scale=None, blocks=None, mass=None, out=None,
                       return_lse=False):
    """Attention of one new token per request over its cached tokens.

    ``q`` [requests, heads, dim] bf16 or fp16, ``kv`` in the same type; head ``h``
    reads key head ``h // (heads // kv_heads)``.  ``scale`` defaults to
    ``dim ** -0.5``.  Returns ``out`` like ``q`` and, with ``return_lse``, the
    natural log-sum-exp of the scaled scores, fp32 [requests, heads] (to join
    it with attention over other tokens).  A request without tokens gets zeros
    and ``-inf``.

    ``blocks`` int32 [requests, kv_heads, n] reads only the listed blocks of a
    request for each key head (what ``paged_kv_select`` returns; entries that are
    no block of the request are skipped, the order does not matter, and a block
    listed twice counts twice; of a row, only as many entries as the request has
    blocks are looked at).

    ``mass`` fp32 [requests, blocks of the table] is added to in place: the
    attention weight that the heads gave to each block, summed over heads and
    tokens, so a request's row grows by ``heads`` in all.  It needs a block size
    that is a multiple of 16 and at most 1024 heads, takes no ``blocks``, and a
    workspace of ``requests * blocks of the table * block / 16 * heads`` fp32 numbers.

    What is not finite in a token that counts shows, and nowhere else: a value that
    is infinite or no number makes that channel of its heads' results infinite or no
    number; a score of minus infinity counts for nothing; one of plus infinity or no
    number makes the head's result, its log-sum and the mass of its request no number.
    Other places of the cache may hold anything.
    """
    return native_kv().attention(q, kv, block_table, context_lens, scale, blocks, mass, out, return_lse)


def paged_kv_bounds(kv, block_table, context_lens, bounds, *, new_tokens=None):
    """Write the key bounds of the requests' pages: ``bounds`` [pages, kv_heads, 2,
    dim], contiguous and in the cache's type, gets the smallest (0) and the largest
    (1) key of each channel over the tokens that the page holds (keys
    that are not a number are passed over).  ``new_tokens`` recomputes only the pages that hold one of the last ``new_tokens`` tokens of
    their request.  Other rows are left as they were; a page that two requests
    share has to be filled alike in both.  Returns ``bounds``.
    """
    native_kv().bounds(kv, block_table, context_lens, bounds, new_tokens)
    return bounds


def paged_kv_select(q, bounds, block_table, context_lens, keep, *, block_size, sink=1, recent=1):
    """The ``keep`` blocks of each request that a key head's group of query heads
    may attend to most: int32 [requests, kv_heads, keep], ascending, -1 behind.

    A block's score is the largest that ``q . k`` could be for a key within the
    block's ``bounds`` (``paged_kv_bounds``), summed over the group's heads:
    ``sum_h sum_d max(q_hd * lo_d, q_hd * hi_d)``, summed in 64 bits and rounded to
    fp32 once.  A channel whose query is 0 adds nothing whatever its bounds are, and of
    two bounds the one that is a number counts.  The first ``sink`` and the last ``recent`` blocks are always
    taken, the others by score, ties to the lowest index; a score that is not a
    number ranks lowest.  ``bounds`` may have more rows than the cache has pages:
    a table of its own then also ranks blocks that are offloaded.  Entries that
    are no row of ``bounds`` are not taken.
    """
    return native_kv().select(q, bounds, block_table, context_lens, keep, block_size, sink, recent)


class KVEviction(NamedTuple):
    """What ``paged_kv_evict`` returns: the requests without the evicted blocks, and those blocks."""

    block_table: object     # int32 [requests, blocks]: kept pages in their order, -1 behind
    context_lens: object    # int32 [requests]: tokens of the kept blocks
    mass: object            # fp32 [requests, blocks]: mass of the kept blocks, 0 behind
    evicted_blocks: object  # int32 [requests, blocks]: pages that leave, in their order, -1 behind
    evicted_index: object   # int32 [requests, blocks]: their places in the old table, -1 behind
    evicted_count: object   # int32 [requests]


def paged_kv_evict(mass, block_table, context_lens, budget, *, block_size, sink=1, recent=1,
                   pages=None) -> KVEviction:
    """Cut every request to at most ``budget`` blocks: the first ``sink`` and the last
    ``recent`` stay, the others by accumulated attention weight (``mass`` of
    ``paged_kv_attention``), ties to the lowest index; mass that is not a number
    ranks lowest.  ``recent`` is at least 1, so the block that is being filled
    stays the last.  Blocks that are not resident take no place in the
    budget, are dropped and not listed: negative table entries, and with ``pages``,
    the cache's number of pages, entries from there on too (without it every other
    entry is taken for a page).  Requests are cut each on its own: a page that two of
    them share may leave one and stay with the other.  The inputs are left as they were.
    """
    return KVEviction(*native_kv().evict(mass, block_table, context_lens, budget, block_size, sink, recent,
                                          pages))


__all__ = ["KVEviction", "paged_kv_attention", "paged_kv_bounds", "paged_kv_evict", "paged_kv_select"]
