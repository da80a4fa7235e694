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

MAX_REQUESTS = 8192
MAX_DIM = 256
MAX_BLOCK = 65536


def _torch():
    import torch

    return torch


def _need(ok: bool, why: str) -> None:
    if not ok:
        raise ValueError(why)


def _int(v, name: str, least: int) -> int:
    _need(isinstance(v, int) and not isinstance(v, bool) and least <= v < 2**31, f"{name} must be an integer >= {least}")
    return v


def _kv_type(dtype):
    torch = _torch()
    if dtype == torch.bfloat16:
        return native().KV_BF16
    if dtype == torch.float16:
        return native().KV_FP16
    raise ValueError("the cache must be bf16 or fp16")


def _cuda(device) -> None:
    _need(device.type == "cuda", "the tensors must be on a CUDA device")


def _no_grad(*tensors) -> None:
    if _torch().is_grad_enabled():
        _need(not any(t.requires_grad for t in tensors), "the paged-KV operators have no gradient: call them under torch.no_grad()")


def _requests(block_table, context_lens, device, block: int):
    """Checked ``KvRequests`` of a table and its lengths."""
    torch = _torch()
    _need(block_table.dim() == 2 and block_table.dtype == torch.int32, "block_table must be int32 [requests, blocks]")
    n, width = block_table.shape
    _need(context_lens.dim() == 1 and context_lens.dtype == torch.int32 and context_lens.shape[0] == n,
          "context_lens must be int32 [requests]")
    _need(block_table.device == device and context_lens.device == device, "all tensors must be on one CUDA device")
    _need(n <= MAX_REQUESTS, f"at most {MAX_REQUESTS} requests")
    _need(block <= MAX_BLOCK, f"at most {MAX_BLOCK} tokens a block")
    _need(width * block <= 2**31 - 2 * MAX_BLOCK, "block_table is too wide: a request has at most 2**31 tokens")
    _need(n * width * block < 2**35, "block_table is too large: at most 2**35 tokens in all")
    _need(width <= 1 or block_table.stride(1) == 1, "block_table's rows must be contiguous")
    _need(n <= 1 or context_lens.stride(0) == 1, "context_lens must be contiguous")
    return native().KvRequests(block_table.data_ptr(), block_table.stride(0), context_lens.data_ptr(), n, width)


def _cache(kv):
    """Checked ``PagedKv`` of a layer's cache."""
    _need(kv.dim() == 5 and kv.shape[0] == 2, "kv must be [2, pages, block, kv_heads, dim]")
    _, pages, block, heads, dim = kv.shape
    kind = _kv_type(kv.dtype)
    _need(heads >= 1 and block >= 1 and dim % 8 == 0 and 8 <= dim <= MAX_DIM,
          f"kv's dim must be a multiple of 8 from 8 to {MAX_DIM}, and it must have heads and tokens")
    _need(pages < 2**31, "too many pages")
    lane, page, token, head, last = kv.stride()
    _need(last == 1, "kv's last dimension must be contiguous")
    _need((kv.data_ptr() | 2 * lane | 2 * page | 2 * token | 2 * head) % 16 == 0,
          "kv's address and strides must be multiples of 16 bytes")
    return native().PagedKv(kv.data_ptr(), lane, page, token, head, pages, block, heads, dim, kind)


def _query(q, device, dtype, dim: int, kv_heads: int, requests: int):
    _need(q.dim() == 3 and q.dtype == dtype and q.device == device,
          "q must be [requests, heads, dim] in the cache's type and on its device")
    _need(q.shape[0] == requests, "q and block_table must have as many requests")
    _need(q.shape[2] == dim and q.shape[1] >= 1 and q.shape[1] % kv_heads == 0,
          "q's dim must be the cache's, and its heads a multiple of the cache's")
    # pairs are loaded at once: a view that splits them is copied
    if q.stride(2) != 1 or (q.data_ptr() | 2 * q.stride(0) | 2 * q.stride(1)) % 4:
        q = q.clone(memory_format=_torch().contiguous_format)
    return q


def _overlap(a, b) -> bool:
    def span(t):
        lo = t.data_ptr()
        return lo, lo + (sum((n - 1) * s for n, s in zip(t.shape, t.stride())) + 1) * t.element_size()

    if not a.numel() or not b.numel():
        return False
    (a0, a1), (b0, b1) = span(a), span(b)
    return a0 < b1 and b0 < a1


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
    that is a multiple of 16 and takes no ``blocks``.
    """
    torch = _torch()
    cache = _cache(kv)
    dev, dim, kv_heads, block = kv.device, kv.shape[4], kv.shape[3], kv.shape[2]
    req = _requests(block_table, context_lens, dev, block)
    n, width = block_table.shape
    q = _query(q, dev, kv.dtype, dim, kv_heads, n)
    _no_grad(q, kv)
    heads = q.shape[1]
    if blocks is not None:
        _need(blocks.dtype == torch.int32 and blocks.device == dev and blocks.dim() == 3 and blocks.is_contiguous()
              and blocks.shape[:2] == (n, kv_heads), "blocks must be contiguous int32 [requests, kv_heads, n]")
    if mass is not None:
        _need(blocks is None, "mass is gathered over all blocks: it takes no blocks=")
        _need(block % 16 == 0, "mass needs a block size that is a multiple of 16")
        _need(mass.dtype == torch.float32 and mass.device == dev and mass.shape == block_table.shape,
              "mass must be fp32 in block_table's shape")
        _need((width <= 1 or mass.stride(1) == 1) and (n <= 1 or mass.stride(0) >= width),
              "mass must have contiguous rows of their own")
    if out is not None:
        _need(out.dtype == q.dtype and out.device == dev and out.shape == q.shape and out.is_contiguous()
              and out.data_ptr() % 4 == 0, "out must be contiguous, like q, on a 4-byte boundary")
        _need(not _overlap(out, q) and not _overlap(out, kv), "out must not overlap q or kv")
    _cuda(dev)
    if out is None:
        out = torch.empty((n, heads, dim), dtype=q.dtype, device=dev)
    lse = torch.empty((n, heads), dtype=torch.float32, device=dev)
    call = native().KvAttention(cache, req, q.data_ptr(), q.stride(0), q.stride(1), heads,
                                dim ** -0.5 if scale is None else float(scale),
                                0 if blocks is None else blocks.data_ptr(), 0 if blocks is None else blocks.shape[2],
                                0 if mass is None else mass.data_ptr(), 0 if mass is None else mass.stride(0))
    if blocks is not None and blocks.shape[2] == 0:
        out.zero_()
        lse.fill_(float("-inf"))
    else:
        work = torch.empty(call.work_bytes(dev.index), dtype=torch.uint8, device=dev)
        call.run(out.data_ptr(), lse.data_ptr(), work.data_ptr(), dev.index, torch.cuda.current_stream(dev).cuda_stream)
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
    cache = _cache(kv)
    req = _requests(block_table, context_lens, kv.device, kv.shape[2])
    _, pages, _, heads, dim = kv.shape
    _no_grad(kv, bounds)
    _need(bounds.dtype == kv.dtype and bounds.device == kv.device and bounds.shape == (pages, heads, 2, dim)
          and bounds.is_contiguous() and bounds.data_ptr() % 16 == 0,
          "bounds must be contiguous [pages, kv_heads, 2, dim] in the cache's type, on a 16-byte boundary")
    _need(not _overlap(bounds, kv), "bounds must not overlap kv")
    since = -1 if new_tokens is None else _int(new_tokens, "new_tokens", 0)
    _cuda(kv.device)
    native().paged_kv_bounds(cache, req, since, bounds.data_ptr(), kv.device.index,
                             torch.cuda.current_stream(kv.device).cuda_stream)
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
    _need(bounds.dim() == 4 and bounds.shape[2] == 2 and bounds.is_contiguous() and bounds.data_ptr() % 16 == 0,
          "bounds must be contiguous [pages, kv_heads, 2, dim] on a 16-byte boundary")
    dev = bounds.device
    pages, kv_heads, _, dim = bounds.shape
    kind = _kv_type(bounds.dtype)
    _need(kv_heads >= 1 and dim % 8 == 0 and 8 <= dim <= MAX_DIM and pages < 2**31,
          f"bounds' dim must be a multiple of 8 from 8 to {MAX_DIM}")
    block = _int(block_size, "block_size", 1)
    req = _requests(block_table, context_lens, dev, block)
    n, width = block_table.shape
    q = _query(q, dev, bounds.dtype, dim, kv_heads, n)
    _no_grad(q, bounds)
    keep, sink, recent = _int(keep, "keep", 1), _int(sink, "sink", 0), _int(recent, "recent", 0)
    _need(sink + recent <= keep, "keep must be at least sink + recent")
    _cuda(dev)
    out = torch.empty((n, kv_heads, keep), dtype=torch.int32, device=dev)
    scores = torch.empty((n, kv_heads, width), dtype=torch.float32, device=dev)
    native().paged_kv_select(req, q.data_ptr(), q.stride(0), q.stride(1), q.shape[1], bounds.data_ptr(), pages, block,
                             kv_heads, dim, kind, keep, sink, recent, scores.data_ptr(), out.data_ptr(), dev.index,
                             torch.cuda.current_stream(dev).cuda_stream)
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
    _need(mass.dtype == torch.float32 and mass.shape == block_table.shape, "mass must be fp32 in block_table's shape")
    dev = mass.device
    block = _int(block_size, "block_size", 1)
    req = _requests(block_table, context_lens, dev, block)
    n, width = mass.shape
    _need(width <= 1 or mass.stride(1) == 1, "mass' rows must be contiguous")
    budget, sink, recent = _int(budget, "budget", 1), _int(sink, "sink", 0), _int(recent, "recent", 1)
    _need(sink + recent <= budget, "budget must be at least sink + recent")
    _cuda(dev)
    e = KVEviction(*(torch.empty(s, dtype=t, device=dev) for s, t in (
        ((n, width), torch.int32), ((n,), torch.int32), ((n, width), torch.float32), ((n, width), torch.int32),
        ((n, width), torch.int32), ((n,), torch.int32))))
    native().paged_kv_evict(req, mass.data_ptr(), mass.stride(0), block, budget, sink, recent,
                            e.block_table.data_ptr(), e.context_lens.data_ptr(), e.mass.data_ptr(),
                            e.evicted_blocks.data_ptr(), e.evicted_index.data_ptr(), e.evicted_count.data_ptr(),
                            dev.index, torch.cuda.current_stream(dev).cuda_stream)
    return e


__all__ = ["KVEviction", "paged_kv_attention", "paged_kv_bounds", "paged_kv_evict", "paged_kv_select"]
