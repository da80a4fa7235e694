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
    both = torch.zeros(1, PAGES, 16, 2, 64, dtype=torch.bfloat16).expand(2, -1, -1, -1, -1)
    for kv in (heads, apart, both):
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


# ---- what leaves, as a whole: room on the host, pages that requests share ---------------------------------


def plain_evict(mass, table, lens, budget, *, block_size, sink=1, recent=1, pages=None):
    """What ``paged_kv_evict`` returns, on the CPU."""
    from tests.paged_kv_cases import best

    rows, width = table.shape
    pages = 2**31 if pages is None else pages
    kept, gone, at = (torch.full((rows, width), -1, dtype=torch.int32) for _ in range(3))
    new_mass, new_lens, count = torch.zeros(rows, width), torch.zeros(rows, dtype=torch.int32), torch.zeros(rows, dtype=torch.int32)
    for b in range(rows):
        n = -(-int(lens[b]) // block_size)
        can = [0 <= int(table[b, j]) < pages for j in range(n)]
        stay = best(mass[b, :n].tolist(), can, budget, sink, recent)
        out = [j for j in range(n) if can[j] and j not in stay]
        kept[b, : len(stay)], new_mass[b, : len(stay)] = table[b, stay], mass[b, stay]
        gone[b, : len(out)], at[b, : len(out)] = table[b, out], torch.tensor(out, dtype=torch.int32)
        new_lens[b], count[b] = sum(min(block_size, int(lens[b]) - j * block_size) for j in stay), len(out)
    return ops.KVEviction(kept, new_lens, new_mass, gone, at, count)


class Recorder(PagedKVOffloader):
    """Records its transfers instead of making them."""

    def __init__(self, kvs):
        super().__init__(Engine(), kvs, target=0, sync_stream=False)
        self.calls = []

    def save(self, block_ids, host_ptr, host_bytes, host_off=0):
        self.calls.append((list(block_ids), host_off))
        return len(block_ids)


def batch():
    table = torch.tensor([[0, 1, 2, 3, 4], [0, 1, 5, 6, -1]], dtype=torch.int32)
    mass = torch.tensor([[9.0, 1.0, 8.0, 2.0, 0.0], [9.0, 1.0, 2.0, 0.0, 0.0]])
    return mass, table, torch.tensor([75, 60], dtype=torch.int32)


def test_room_for_all_that_leaves_is_checked_before_the_first_transfer(monkeypatch):
    monkeypatch.setattr(ops, "paged_kv_evict", plain_evict)
    store = Recorder([cache()])
    need = store.prefix_bytes(2) + store.prefix_bytes(1)
    for room, off in ((need - 1, 0), (need + 63, 64), (0, 0), (1 << 20, -16)):
        with pytest.raises(ValueError, match="host region"):
            store.evict(*batch(), 3, 4096, room, block_size=16, host_off=off)
    assert store.calls == []
    e, gone = store.evict(*batch(), 3, 4096, need + 64, block_size=16, host_off=64)
    assert store.calls == [([1, 3], 64), ([1], 64 + store.prefix_bytes(2))] and len(gone) == 2
    store.evict(*batch(), 5, 4096, 0, block_size=16)  # nothing leaves: no room is needed


def daemon_offloader(kvs):
    from test_daemon_landing import node

    from pcie_pool_b200 import TurboBusClient
    from pcie_pool_b200.adapters.kv_offload import DaemonKVOffloader

    _, dc, sid, _ = node()
    return DaemonKVOffloader(TurboBusClient(daemon=dc), dc, session_id=sid, job_id="job", kv_caches=kvs, units_per_chunk=4,
                             sync_stream=False)


def test_blocks_leave_through_the_daemon_and_come_back(monkeypatch):
    """The mock world moves real bytes: two layers are cut, what left is saved, overwritten, and restored elsewhere."""
    monkeypatch.setattr(ops, "paged_kv_evict", plain_evict)
    g = torch.Generator().manual_seed(5)
    kvs = [torch.randn(2, 16, 16, 2, 16, generator=g).to(torch.bfloat16) for _ in range(2)]
    store = daemon_offloader(kvs)
    mass, table, lens = batch()
    table[1, 1], table[1, 3] = 16, 7                # an entry that is no page of the cache; no page is shared
    table[1, 0] = 8
    small = torch.zeros(store.prefix_bytes(3) - 1, dtype=torch.uint8)
    with pytest.raises(ValueError, match="host region"):
        store.evict(mass, table, lens, 2, small, block_size=16)
    host = torch.zeros(store.prefix_bytes(4), dtype=torch.uint8)
    e, gone = store.evict(mass, table, lens, 2, host, block_size=16)
    assert [(x.request, x.blocks, x.index) for x in gone] == [(0, [1, 2, 3], [1, 2, 3]), (1, [5], [2])]
    before = [kv.clone() for kv in kvs]
    for kv in kvs:
        kv[:, [1, 2, 3, 5]] = 0
    for x, pages in zip(gone, ([12, 10, 15], [11])):
        store.restore(pages, host, host_off=x.host_off)
        for kv, old in zip(kvs, before):
            assert torch.equal(kv[:, pages], old[:, x.blocks])


def test_pages_that_requests_share_are_free_once_nobody_keeps_them(monkeypatch):
    monkeypatch.setattr(ops, "paged_kv_evict", plain_evict)
    # page 1: both lose it; page 2: the first keeps it, the second loses it; page 4 stands twice in one row and leaves twice
    table = torch.tensor([[0, 1, 2, 3, 9], [0, 1, 2, 6, 9], [4, 5, 4, 7, 8]], dtype=torch.int32)
    mass = torch.tensor([[9.0, 1.0, 8.0, 2.0, 0.0], [9.0, 1.0, 2.0, 5.0, 0.0], [1.0, 9.0, 1.0, 8.0, 0.0]])
    store = Recorder([torch.zeros(2, 16, 16, 2, 64, dtype=torch.bfloat16)])
    e, gone = store.evict(mass, table, torch.tensor([80, 80, 80], dtype=torch.int32), 3, 4096, 1 << 20, block_size=16, sink=0)
    assert e.block_table[:, :3].tolist() == [[0, 2, 9], [0, 6, 9], [5, 7, 8]]
    assert [(x.blocks, x.free) for x in gone] == [([1, 3], [1, 3]), ([1, 2], []), ([4, 4], [4])]
    # every request has all its blocks on the host, in a region of its own
    assert [c[0] for c in store.calls] == [[1, 3], [1, 2], [4, 4]]
    assert [c[1] for c in store.calls] == [0, store.prefix_bytes(2), store.prefix_bytes(4)]


# ---- what the operators write to -------------------------------------------------------------------------


@pytest.fixture
def good():
    from tests.paged_kv_cases import make

    q, kv, table, lens = make(0, [20, 5], 16, 8, 2, 64, torch.bfloat16)
    return dict(q=q, kv=kv, block_table=table, context_lens=lens)


@pytest.mark.parametrize("name", ["mass", "out", "kv", "q"])
def test_attention_refuses_what_requires_a_gradient(good, name):
    """mass and out are written in place: autograd would not see it."""
    given = dict(good, mass=torch.zeros(good["block_table"].shape), out=torch.empty_like(good["q"]))
    given[name] = given[name].clone().requires_grad_()
    with pytest.raises(ValueError, match="no gradient"):
        ops.paged_kv_attention(**given)
    with torch.no_grad(), pytest.raises(ValueError, match="CUDA device"):
        ops.paged_kv_attention(**given)


def shared(dtype, shape, with_shape, with_dtype, at=0):
    """Two tensors in one buffer: the second begins `at` bytes behind the first."""
    buf = torch.zeros(1 << 16, dtype=torch.uint8)
    one, two = (torch.empty(s, dtype=t) for s, t in ((shape, dtype), (with_shape, with_dtype)))
    size = [x.numel() * x.element_size() for x in (one, two)]
    return (buf[: size[0]].view(dtype).view(shape), buf[at: at + size[1]].view(with_dtype).view(with_shape))


@pytest.mark.parametrize("written,read", [("out", "block_table"), ("out", "context_lens"), ("out", "blocks"), ("out", "mass"),
                                          ("mass", "q"), ("mass", "kv"), ("mass", "block_table"), ("mass", "context_lens"),
                                          ("bounds", "block_table"), ("bounds", "context_lens")])
def test_what_is_written_must_not_share_memory_with_what_is_read(good, written, read):
    kv = good["kv"][:, :3].contiguous()
    args = dict(good, kv=kv, blocks=torch.zeros(2, 2, 1, dtype=torch.int32), mass=torch.zeros(good["block_table"].shape),
                out=torch.empty_like(good["q"]), bounds=torch.zeros(3, 2, 2, 64, dtype=kv.dtype))
    args.pop("mass" if "blocks" in (written, read) else "blocks")  # they do not go together
    w, r = args[written], args[read]
    args[written], args[read] = shared(w.dtype, w.shape, r.shape, r.dtype)
    if written == "bounds":
        with pytest.raises(ValueError, match="must not overlap"):
            ops.paged_kv_bounds(args["kv"], args["block_table"], args["context_lens"], args["bounds"])
        return
    args.pop("bounds")
    with pytest.raises(ValueError, match="must not overlap"):
        ops.paged_kv_attention(**args)


def test_neighbours_in_one_buffer_do_not_overlap(good):
    width = good["block_table"].shape[1]
    rows = torch.zeros(2, 4 * width, dtype=torch.int32)   # table and mass side by side, in both orders, and behind each other
    for first, second in ((0, 1), (1, 0), (3, 2), (0, 3)):
        table = rows[:, first * width: (first + 1) * width].copy_(good["block_table"])
        mass = rows.view(torch.float32)[:, second * width: (second + 1) * width]
        with pytest.raises(ValueError, match="CUDA device"):
            ops.paged_kv_attention(**dict(good, block_table=table), mass=mass)
    for off in (1, width - 1):                            # a column in common
        with pytest.raises(ValueError, match="must not overlap"):
            ops.paged_kv_attention(**dict(good, block_table=rows[:, width: 2 * width]),
                                   mass=rows.view(torch.float32)[:, width + off: 2 * width + off])
        with pytest.raises(ValueError, match="must not overlap"):
            ops.paged_kv_attention(**dict(good, block_table=rows[:, width: 2 * width]),
                                   mass=rows.view(torch.float32)[:, width - off: 2 * width - off])
    out, mass = shared(good["q"].dtype, good["q"].shape, (2, width), torch.float32, at=good["q"].numel() * 2)
    with pytest.raises(ValueError, match="CUDA device"):
        ops.paged_kv_attention(**good, out=out, mass=mass)


def test_strides_of_dimensions_of_one_do_not_count():
    """A cache of one page, one head or one token a page: torch gives such a dimension any stride."""
    flat = torch.zeros(1 << 14, dtype=torch.bfloat16)
    q, table, lens = torch.zeros(1, 4, 64, dtype=torch.bfloat16), torch.zeros(1, 1, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    sizes, strides = [2, 4, 16, 2, 64], [4096, 1024, 64, 2048, 1]
    for i in (1, 2, 3):
        one = [1 if j == i else n for j, n in enumerate(sizes)]
        odd = [3 if j == i else n for j, n in enumerate(strides)]
        kv = flat.as_strided(one, odd)
        with pytest.raises(ValueError, match="CUDA device"):
            ops.paged_kv_attention(q, kv, table, lens)
        with pytest.raises(ValueError, match="multiples of 16 bytes"):
            ops.paged_kv_attention(q, flat.as_strided(sizes, odd), table, lens)


def test_what_a_request_has_may_lie_in_one_row(good):
    """A row a request: its query, its mass and its table next to each other."""
    n, width = good["block_table"].shape
    rows = torch.zeros(n, 8 * 64 * 2 + 4 * width + 4 * width + 16, dtype=torch.uint8)
    q = rows[:, : 8 * 64 * 2].view(torch.bfloat16).unflatten(1, (8, 64)).copy_(good["q"])
    at = 8 * 64 * 2
    mass = rows[:, at: at + 4 * width].view(torch.float32)
    table = rows[:, at + 4 * width: at + 8 * width].view(torch.int32).copy_(good["block_table"])
    assert not q.is_contiguous() and q.data_ptr() == rows.data_ptr()
    with pytest.raises(ValueError, match="CUDA device"):
        ops.paged_kv_attention(**dict(good, q=q, block_table=table), mass=mass)
    for off in (-4, 4):
        with pytest.raises(ValueError, match="must not overlap"):
            ops.paged_kv_attention(**dict(good, q=q, block_table=table), mass=rows[:, at + off: at + off + 4 * width].view(torch.float32))
