"""Operators on the paged KV cache of one layer: attention of one new token per
request, the key bounds of the cache's pages, the blocks that sparse attention
reads, and the blocks that may leave the GPU.

The cache is the layer tensor that ``paged_kv_gather`` takes: ``[2, pages,
block, kv_heads, dim]``, K then V, in any strides that are multiples of 16 bytes
with a contiguous last dimension; a ``[pages, 2, ...]`` cache is passed as
``kv.transpose(0, 1)``.  Request ``b`` holds ``context_lens[b]`` tokens, block
``j`` of it in page ``block_table[b, j]``.  A table entry that is no page
(negative, or ``>= pages``) is a block that is not resident -- offloaded, say --
and its tokens are left out.  Lengths and tables are read on the device when the
kernel runs, so all calls can be captured into a CUDA graph and replayed with
other contents.

A serving step with a bounded cache strings them together::

    out = paged_kv_attention(q, kv, table, lens, mass=mass)          # every layer adds to mass
    e = paged_kv_evict(mass, table, lens, budget, block_size=16)     # pages e.evicted_blocks leave
    # PagedKVOffloader.save(...) them, then go on with e.block_table, e.context_lens, e.mass

and one with sparse reads::

    paged_kv_bounds(kv, table, lens, bounds, new_tokens=1)
    blocks = paged_kv_select(q, bounds, table, lens, keep, block_size=16)
    out = paged_kv_attention(q, kv, table, lens, blocks=blocks)

All run on the tensors' device and its current stream, without a synchronisation,
and raise ``ValueError`` for what they do not take; none has a gradient.
"""

from __future__ import annotations

from typing import NamedTuple

from .._native import native

MAX_REQUESTS = 4096
MAX_DIM = 256
MAX_BLOCK = 65536
MAX_MASS_HEADS = 1024


def _torch():
    import torch

    return torch


def _int(v, name: str, least: int) -> int:
    if not isinstance(v, int) or isinstance(v, bool) or not least <= v < 2**31:
        raise ValueError(f"{name} must be an integer >= {least}")
    return v


def _kv_type(dtype, torch) -> int:
    if dtype == torch.bfloat16:
        return 0
    if dtype == torch.float16:
        return 1
    raise ValueError("the cache must be bf16 or fp16")


def _runs(torch, *tensors) -> int:
    """The stream that a call on these tensors runs on, as an integer; the last check of every call."""
    for t in tensors:
        if t.requires_grad and torch.is_grad_enabled():
            raise ValueError("the paged-KV operators have no gradient: call them under torch.no_grad()")
    t = tensors[0]
    if not t.is_cuda:
        raise ValueError("the tensors must be on a CUDA device")
    # current_stream(t.device).cuda_stream without the Stream object: a tenth of the call's host time
    return torch._C._cuda_getCurrentRawStream(t.get_device())


def _requests(torch, block_table, context_lens, device: int, block: int):
    """Checks a table and its lengths; the arguments that describe them to the native call."""
    if block_table.dtype != torch.int32 or block_table.dim() != 2:
        raise ValueError("block_table must be int32 [requests, blocks]")
    n, width = block_table.shape
    if n > MAX_REQUESTS:
        raise ValueError(f"at most {MAX_REQUESTS} requests")
    if context_lens.dtype != torch.int32 or context_lens.shape != (n,):
        raise ValueError("context_lens must be int32 [requests]")
    if block_table.get_device() != device or context_lens.get_device() != device:
        raise ValueError("all tensors must be on one CUDA device")
    row, col = block_table.stride()
    if block > MAX_BLOCK:
        raise ValueError(f"at most {MAX_BLOCK} tokens a block")
    if width * block > 2**31 - 2 * MAX_BLOCK:
        raise ValueError("block_table is too wide: a request has at most 2**31 tokens")
    if n * width * block >= 2**34:
        raise ValueError("block_table is too large: at most 2**34 tokens in all")
    if col != 1 and width > 1:
        raise ValueError("block_table's rows must be contiguous")
    if n > 1 and not context_lens.is_contiguous():
        raise ValueError("context_lens must be contiguous")
    return block_table.data_ptr(), row, context_lens.data_ptr(), n, width


def _cache(torch, kv):
    """Checks a layer's cache; the arguments that describe it to the native call."""
    if kv.dim() != 5 or kv.shape[0] != 2:
        raise ValueError("kv must be [2, pages, block, kv_heads, dim]")
    kind = _kv_type(kv.dtype, torch)
    _, pages, block, heads, dim = kv.shape
    lane, page, token, head, last = kv.stride()
    at = kv.data_ptr()
    if dim % 8 or not 8 <= dim <= MAX_DIM or heads < 1 or block < 1:
        raise ValueError(f"kv's dim must be a multiple of 8 from 8 to {MAX_DIM}, and it must have heads and tokens")
    if pages >= 2**31:
        raise ValueError("too many pages")
    if last != 1:
        raise ValueError("kv's last dimension must be contiguous")
    if at % 16 or (lane | page | token | head) % 8:
        raise ValueError("kv's address and strides must be multiples of 16 bytes")
    return at, lane, page, token, head, pages, block, heads, dim, kind


def _query(torch, q, device: int, dtype, dim: int, kv_heads: int, requests: int):
    """Checks the queries; pairs are loaded at once, so a view that splits them is copied."""
    if q.dim() != 3 or q.dtype != dtype or q.get_device() != device:
        raise ValueError("q must be [requests, heads, dim] in the cache's type and on its device")
    n, heads, d = q.shape
    if n != requests:
        raise ValueError("q and block_table must have as many requests")
    if d != dim or heads < 1 or heads % kv_heads:
        raise ValueError("q's dim must be the cache's, and its heads a multiple of the cache's")
    row, head, last = q.stride()
    at = q.data_ptr()
    if last != 1 or at % 4 or (row | head) % 2:
        q = q.clone(memory_format=torch.contiguous_format)
        at, row, head = q.data_ptr(), heads * dim, dim
    return q, (at, row, head, heads)


def _overlap(t, cache) -> bool:
    """Whether a contiguous 16-bit tensor shares memory with the span of a cache (its arguments)."""
    at, lane, page, token, head, pages, block, heads, dim, _ = cache
    end = at + 2 * (lane + max(pages - 1, 0) * page + (block - 1) * token + (heads - 1) * head + dim)
    low = t.data_ptr()
    return low < end and at < low + 2 * t.numel()


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
    that is a multiple of 16 and at most 1024 heads, and takes no ``blocks``.
    """
    torch = _torch()
    cache = _cache(torch, kv)
    pages, block, kv_heads, dim = cache[5:9]
    dev, index = kv.device, kv.get_device()
    req = _requests(torch, block_table, context_lens, index, block)
    n, width = req[3:]
    q, query = _query(torch, q, index, kv.dtype, dim, kv_heads, n)
    heads = query[3]
    listed = weights = (0, 0)
    if blocks is not None:
        if (blocks.dtype != torch.int32 or blocks.get_device() != index or blocks.dim() != 3 or not blocks.is_contiguous()
                or blocks.shape[:2] != (n, kv_heads)):
            raise ValueError("blocks must be contiguous int32 [requests, kv_heads, n]")
        listed = blocks.data_ptr(), blocks.shape[2]
    if mass is not None:
        if blocks is not None:
            raise ValueError("mass is gathered over all blocks: it takes no blocks=")
        if heads > MAX_MASS_HEADS:
            raise ValueError(f"mass takes at most {MAX_MASS_HEADS} heads")
        if block % 16:
            raise ValueError("mass needs a block size that is a multiple of 16")
        if mass.dtype != torch.float32 or mass.get_device() != index or mass.shape != block_table.shape:
            raise ValueError("mass must be fp32 in block_table's shape")
        row, col = mass.stride()
        if (width > 1 and col != 1) or (n > 1 and row < width):
            raise ValueError("mass must have contiguous rows of their own")
        weights = mass.data_ptr(), row
    if out is not None:
        if (out.dtype != q.dtype or out.get_device() != index or out.shape != q.shape or not out.is_contiguous()
                or out.data_ptr() % 4):
            raise ValueError("out must be contiguous, like q, on a 4-byte boundary")
        at, row, head, _ = query
        size = 2 * (max(n - 1, 0) * row + (heads - 1) * head + dim)
        if _overlap(out, cache) or (out.data_ptr() < at + size and at < out.data_ptr() + out.numel() * 2):
            raise ValueError("out must not overlap q or kv")
    stream = _runs(torch, kv, q)
    if out is None:
        out = torch.empty_like(q) if q.is_contiguous() else q.new_empty(q.shape)
    lse = q.new_empty((n, heads), dtype=torch.float32)
    if blocks is not None and listed[1] == 0:
        out.zero_()
        lse.fill_(float("-inf"))
    else:
        C = native()
        work = torch.empty(C.paged_kv_attention_work(n, width, block, heads, kv_heads, dim, mass is not None, index),
                           dtype=torch.uint8, device=dev)
        C.paged_kv_attention(*cache, *req, *query, dim ** -0.5 if scale is None else float(scale), *listed, *weights,
                             out.data_ptr(), lse.data_ptr(), work.data_ptr(), index, stream)
    return (out, lse) if return_lse else out


def paged_kv_bounds(kv, block_table, context_lens, bounds, *, new_tokens=None):
    """Write the key bounds of the requests' pages: ``bounds`` [pages, kv_heads, 2,
    dim], contiguous and in the cache's type, gets the smallest (0) and the largest
    (1) key of each channel over the tokens that the page holds (keys
    that are not a number are passed over).  ``new_tokens`` recomputes only the pages that hold one of the last ``new_tokens`` tokens of
    their request.  Other rows are left as they were; a page that two requests
    share has to be filled alike in both.  Returns ``bounds``.
    """
    torch = _torch()
    cache = _cache(torch, kv)
    pages, block, heads, dim = cache[5:9]
    index = kv.get_device()
    req = _requests(torch, block_table, context_lens, index, block)
    if (bounds.dtype != kv.dtype or bounds.get_device() != index or bounds.shape != (pages, heads, 2, dim)
            or not bounds.is_contiguous() or bounds.data_ptr() % 16):
        raise ValueError("bounds must be contiguous [pages, kv_heads, 2, dim] in the cache's type, on a 16-byte boundary")
    if _overlap(bounds, cache):
        raise ValueError("bounds must not overlap kv")
    since = -1 if new_tokens is None else _int(new_tokens, "new_tokens", 0)
    stream = _runs(torch, kv, bounds)
    native().paged_kv_bounds(*cache, *req, since, bounds.data_ptr(), index, stream)
    return bounds


def paged_kv_select(q, bounds, block_table, context_lens, keep, *, block_size, sink=1, recent=1):
    """The ``keep`` blocks of each request that a key head's group of query heads
    may attend to most: int32 [requests, kv_heads, keep], ascending, -1 behind.

    A block's score is the largest that ``q . k`` could be for a key within the
    block's ``bounds`` (``paged_kv_bounds``), summed over the group's heads:
    ``sum_h sum_d max(q_hd * lo_d, q_hd * hi_d)``, summed in 64 bits and rounded to
    fp32 once.  The first ``sink`` and the last ``recent`` blocks are always
    taken, the others by score, ties to the lowest index; a score that is not a
    number ranks lowest.  ``bounds`` may have more rows than the cache has pages:
    a table of its own then also ranks blocks that are offloaded.  Entries that
    are no row of ``bounds`` are not taken.
    """
    torch = _torch()
    if bounds.dim() != 4 or bounds.shape[2] != 2 or not bounds.is_contiguous() or bounds.data_ptr() % 16:
        raise ValueError("bounds must be contiguous [pages, kv_heads, 2, dim] on a 16-byte boundary")
    pages, kv_heads, _, dim = bounds.shape
    index = bounds.get_device()
    kind = _kv_type(bounds.dtype, torch)
    if kv_heads < 1 or dim % 8 or not 8 <= dim <= MAX_DIM or pages >= 2**31:
        raise ValueError(f"bounds' dim must be a multiple of 8 from 8 to {MAX_DIM}")
    block = _int(block_size, "block_size", 1)
    req = _requests(torch, block_table, context_lens, index, block)
    n, width = req[3:]
    q, query = _query(torch, q, index, bounds.dtype, dim, kv_heads, n)
    keep, sink, recent = _int(keep, "keep", 1), _int(sink, "sink", 0), _int(recent, "recent", 0)
    if sink + recent > keep:
        raise ValueError("keep must be at least sink + recent")
    stream = _runs(torch, bounds, q)
    out = block_table.new_empty((n, kv_heads, keep))
    scores = torch.empty(n * kv_heads * width, dtype=torch.float32, device=bounds.device)
    native().paged_kv_select(*req, *query, bounds.data_ptr(), pages, block, kv_heads, dim, kind, keep, sink, recent,
                             scores.data_ptr(), out.data_ptr(), index, stream)
    return out


class KVEviction(NamedTuple):
    """What ``paged_kv_evict`` returns: the requests without the evicted blocks, and those blocks."""

    block_table: object     # int32 [requests, blocks]: kept pages in their order, -1 behind
    context_lens: object    # int32 [requests]: tokens of the kept blocks
    mass: object            # fp32 [requests, blocks]: mass of the kept blocks, 0 behind
    evicted_blocks: object  # int32 [requests, blocks]: pages that leave, in their order, -1 behind
    evicted_index: object   # int32 [requests, blocks]: their places in the old table, -1 behind
    evicted_count: object   # int32 [requests]


def paged_kv_evict(mass, block_table, context_lens, budget, *, block_size, sink=1, recent=1) -> KVEviction:
    """Cut every request to at most ``budget`` blocks: the first ``sink`` and the last
    ``recent`` stay, the others by accumulated attention weight (``mass`` of
    ``paged_kv_attention``), ties to the lowest index; mass that is not a number
    ranks lowest.  ``recent`` is at least 1, so the block that is being filled
    stays the last.  Negative table entries (blocks that are not resident) are
    dropped and not listed.  The inputs are left as they were.
    """
    torch = _torch()
    if mass.dtype != torch.float32 or mass.shape != block_table.shape:
        raise ValueError("mass must be fp32 in block_table's shape")
    index = mass.get_device()
    block = _int(block_size, "block_size", 1)
    req = _requests(torch, block_table, context_lens, index, block)
    n, width = req[3:]
    row, col = mass.stride()
    if width > 1 and col != 1:
        raise ValueError("mass' rows must be contiguous")
    budget, sink, recent = _int(budget, "budget", 1), _int(sink, "sink", 0), _int(recent, "recent", 1)
    if sink + recent > budget:
        raise ValueError("budget must be at least sink + recent")
    stream = _runs(torch, mass)
    # two allocations: an allocation costs as much host time as the launch
    table, pages, places, kept = block_table.new_empty((4, n, width)).unbind(0)
    lens, count = context_lens.new_empty((2, n)).unbind(0)
    kept = kept.view(torch.float32)
    native().paged_kv_evict(*req, mass.data_ptr(), row, block, budget, sink, recent, table.data_ptr(), lens.data_ptr(),
                            kept.data_ptr(), pages.data_ptr(), places.data_ptr(), count.data_ptr(), index, stream)
    return KVEviction(table, lens, kept, pages, places, count)


__all__ = ["KVEviction", "paged_kv_attention", "paged_kv_bounds", "paged_kv_evict", "paged_kv_select"]
