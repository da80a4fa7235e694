"""Pages of the paged KV cache on the host's side, on CPU: ids that are no page of the cache, pages that requests
share, and the room that an eviction needs."""

import pytest
import torch

from pcie_pool_b200 import ops
from pcie_pool_b200.adapters import PagedKVOffloader
from pcie_pool_b200.adapters.vllm import block_table_units

PAGES = 8


class Engine:
    """Stands for the pool engine: no transfer may reach it."""

    def run(self, *args, **more):
        raise AssertionError("a transfer was started")


def cache(pages_first=False):
    shape = (PAGES, 2, 16, 2, 64) if pages_first else (2, PAGES, 16, 2, 64)
    return torch.zeros(shape, dtype=torch.bfloat16)


# ---- ids outside the cache ----------------------------------------------------------------


@pytest.mark.parametrize("pages_first", [False, True])
@pytest.mark.parametrize("ids", [[PAGES], [3, 1000], [-1], [0, -7, 2], [2**31 - 1]])
def test_ids_outside_the_cache_get_no_address(pages_first, ids):
    kvs = [cache(pages_first) for _ in range(2)]
    with pytest.raises(ValueError, match="outside the kv cache"):
        block_table_units(kvs, ids)
    store = PagedKVOffloader(Engine(), kvs, target=0, sync_stream=False)
    with pytest.raises(ValueError, match="outside the kv cache"):
        store.save(ids, 4096, 1 << 30)
    with pytest.raises(ValueError, match="outside the kv cache"):
        store.restore(ids, 4096, 1 << 30)


@pytest.mark.parametrize("ids", [[PAGES], [-1, 0]])
def test_gather_and_scatter_refuse_ids_outside_the_cache(ids):
    with pytest.raises(ValueError, match="outside the kv cache"):
        ops.paged_kv_gather(cache(), ids)
    with pytest.raises(ValueError, match="outside the kv cache"):
        ops.paged_kv_scatter(cache(), ids, torch.zeros(1 << 16, dtype=torch.uint8))


def test_ids_of_the_cache_are_taken():
    kvs = [cache(), cache()]
    addrs, unit = block_table_units(kvs, [PAGES - 1, 0])
    last = kvs[1].data_ptr() + kvs[1].numel() * 2 - unit
    assert last in addrs.tolist() and int(addrs.min()) >= min(kv.data_ptr() for kv in kvs)
    assert block_table_units(kvs, [])[0].size == 0


# ---- views whose K and V lie next to each other ------------------------------------------------


def test_a_transposed_cache_is_no_cache_of_planes():
    """Its units would be two lanes long: the last one ends past the cache, the others cover the next block's keys."""
    view = cache(pages_first=True).transpose(0, 1)
    with pytest.raises(ValueError, match="next to each other"):
        block_table_units([view], [0])
    with pytest.raises(ValueError, match="next to each other"):
        PagedKVOffloader(Engine(), [view], target=0)
    with pytest.raises(ValueError, match="next to each other"):
        ops.paged_kv_gather(view, [0])
    with pytest.raises(ValueError, match="next to each other"):
        ops.paged_kv_scatter(view, [0], torch.zeros(1 << 16, dtype=torch.uint8))


def test_planes_of_any_inner_order_are_taken():
    heads = torch.zeros(2, PAGES, 2, 16, 64, dtype=torch.bfloat16).transpose(2, 3)
    apart = torch.zeros(2, PAGES + 3, 16, 2, 64, dtype=torch.bfloat16)[:, 2: 2 + PAGES]
    for kv in (heads, apart):
        addrs, unit = block_table_units([kv], range(PAGES))
        assert unit == 16 * 2 * 64 * 2 and addrs[-1] == kv.data_ptr() + kv.stride(0) * 2 + (PAGES - 1) * unit


# ---- eviction and the cache's number of pages ---------------------------------------------------------


def test_offloaders_tell_the_eviction_how_many_pages_there_are(monkeypatch):
    asked = []

    def evict(*args, **more):
        asked.append(more)
        none = torch.full((1, 2), -1, dtype=torch.int32)
        return ops.KVEviction(none, None, None, none, none, torch.zeros(1, dtype=torch.int32))

    monkeypatch.setattr(ops, "paged_kv_evict", evict)
    for kvs in ([cache(), cache()], [cache(pages_first=True)]):
        PagedKVOffloader(Engine(), kvs, target=0).evict(None, None, None, 3, 4096, 1 << 20, block_size=16)
    assert [a["pages"] for a in asked] == [PAGES, PAGES]


def test_evict_refuses_numbers_of_pages_that_are_none():
    table = torch.zeros(1, 4, dtype=torch.int32)
    lens = torch.tensor([50], dtype=torch.int32)
    for pages in (-1, 8.0, True, 2**31):
        with pytest.raises(ValueError, match="pages must be"):
            ops.paged_kv_evict(torch.zeros(1, 4), table, lens, 3, block_size=16, pages=pages)
    with pytest.raises(ValueError, match="CUDA device"):
        ops.paged_kv_evict(torch.zeros(1, 4), table, lens, 3, block_size=16, pages=8)


# ---- numbers that 32 bits do not hold ------------------------------------------------------------------


@pytest.mark.parametrize("requests,kv_heads,width", [(4096, 2**20, 1), (4096, 2**19, 1), (4095, 2**20 + 1, 4), (1, 2**20, 2**15),
                                                     (4096, 2**12, 2**13)])
def test_select_refuses_more_rows_than_a_grid_holds(requests, kv_heads, width):
    """4096 requests of 2**20 key heads were 2**32 rows, 0 in 32 bits: nothing was written to the result."""
    q = torch.zeros(1, 1, 8, dtype=torch.bfloat16).expand(requests, kv_heads, 8)
    bounds = torch.zeros(0, kv_heads, 2, 8, dtype=torch.bfloat16)
    table = torch.zeros(1, 1, dtype=torch.int32).expand(requests, width)
    table = table if width == 1 else torch.zeros(1, width, dtype=torch.int32).expand(requests, width)
    with pytest.raises(ValueError, match="too many key heads"):
        ops.paged_kv_select(q, bounds, table, torch.zeros(requests, dtype=torch.int32), 1, block_size=16, recent=0)


def test_select_takes_many_key_heads():
    q = torch.zeros(1, 1, 8, dtype=torch.bfloat16).expand(2047, 2**20, 8)
    bounds = torch.zeros(0, 2**20, 2, 8, dtype=torch.bfloat16)
    table = torch.zeros(1, 1, dtype=torch.int32).expand(2047, 1)
    with pytest.raises(ValueError, match="CUDA device"):
        ops.paged_kv_select(q, bounds, table, torch.zeros(2047, dtype=torch.int32), 1, block_size=16, recent=0)
