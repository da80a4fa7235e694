"""What the paged-KV operators refuse, before anything runs on a GPU: the checks
come in an order that ends with the device, so CPU tensors reach each of them."""

import pytest
import torch

from pcie_pool_b200 import ops
from tests.paged_kv_cases import make


@pytest.fixture
def good():
    q, kv, table, lens = make(0, [20, 5], 16, 8, 2, 64, torch.bfloat16)
    return dict(q=q, kv=kv, block_table=table, context_lens=lens)


def attend(good, **change):
    a = {**good, **change}
    return ops.paged_kv_attention(a.pop("q"), a.pop("kv"), a.pop("block_table"), a.pop("context_lens"), **a)


def wide(t):
    return torch.stack((t, t), -1)[..., 0]


BAD_ATTENTION = {
    "q dims": (lambda a: dict(q=a["q"][0]), "q must be"),
    "q type": (lambda a: dict(q=a["q"].float()), "q must be"),
    "q requests": (lambda a: dict(q=a["q"][:1]), "as many requests"),
    "q dim": (lambda a: dict(q=a["q"][..., :32]), "q's dim"),
    "q heads": (lambda a: dict(q=a["q"][:, :5]), "multiple of the cache's"),
    "no heads": (lambda a: dict(q=a["q"][:, :0]), "multiple of the cache's"),
    "kv dims": (lambda a: dict(kv=a["kv"][0]), "kv must be"),
    "kv planes": (lambda a: dict(kv=a["kv"].transpose(0, 1)), "kv must be"),
    "kv type": (lambda a: dict(kv=a["kv"].float(), q=a["q"].float()), "bf16 or fp16"),
    "kv dim": (lambda a: dict(kv=a["kv"][..., :36]), "multiple of 8"),
    "kv dim large": (lambda a: dict(kv=torch.zeros(2, 4, 16, 2, 264, dtype=torch.bfloat16)), "multiple of 8"),
    "kv order": (lambda a: dict(kv=wide(a["kv"])), "contiguous"),
    "kv address": (lambda a: dict(kv=torch.zeros(8200, dtype=torch.bfloat16)[1:8193].view(2, 2, 16, 2, 64)), "16 bytes"),
    "kv stride": (lambda a: dict(kv=torch.zeros(2, 4, 16, 2, 68, dtype=torch.bfloat16)[..., :64]), "16 bytes"),
    "table dims": (lambda a: dict(block_table=a["block_table"][0]), "block_table must be"),
    "table type": (lambda a: dict(block_table=a["block_table"].long()), "block_table must be"),
    "table order": (lambda a: dict(block_table=wide(a["block_table"])), "rows must be contiguous"),
    "lens type": (lambda a: dict(context_lens=a["context_lens"].long()), "context_lens must be"),
    "lens number": (lambda a: dict(context_lens=a["context_lens"][:1]), "context_lens must be"),
    "lens order": (lambda a: dict(context_lens=wide(a["context_lens"])), "context_lens must be contiguous"),
    "mass type": (lambda a: dict(mass=torch.zeros(a["block_table"].shape, dtype=torch.float64)), "mass must be"),
    "mass shape": (lambda a: dict(mass=torch.zeros(2, 1)), "mass must be"),
    "mass rows": (lambda a: dict(mass=torch.zeros(1, a["block_table"].shape[1]).expand(2, -1)), "rows of their own"),
    "mass heads": (lambda a: dict(q=a["q"][:, :1].expand(-1, 1026, -1), mass=torch.zeros(a["block_table"].shape)), "at most 1024"),
    "mass and blocks": (lambda a: dict(mass=torch.zeros(a["block_table"].shape),
                                       blocks=torch.zeros(2, 2, 1, dtype=torch.int32)), "takes no blocks"),
    "blocks type": (lambda a: dict(blocks=torch.zeros(2, 2, 1, dtype=torch.int64)), "blocks must be"),
    "blocks shape": (lambda a: dict(blocks=torch.zeros(2, 1, 1, dtype=torch.int32)), "blocks must be"),
    "out type": (lambda a: dict(out=torch.zeros(a["q"].shape)), "out must be"),
    "out order": (lambda a: dict(out=wide(a["q"])), "out must be"),
    "out address": (lambda a: dict(out=torch.zeros(2 * 8 * 64 + 1, dtype=torch.bfloat16)[1:].view(2, 8, 64)), "4-byte"),
    "out is q": (lambda a: dict(out=a["q"]), "overlap"),
    "gradient": (lambda a: dict(q=a["q"].clone().requires_grad_()), "no gradient"),
    "device": (lambda a: {}, "CUDA device"),
}


@pytest.mark.parametrize("case", BAD_ATTENTION)
def test_attention_refuses(good, case):
    change, why = BAD_ATTENTION[case]
    with pytest.raises(ValueError, match=why):
        attend(good, **change(good))


def test_attention_refuses_mass_of_odd_blocks():
    q, kv, table, lens = make(0, [20], 24, 4, 2, 64, torch.float16)
    with pytest.raises(ValueError, match="multiple of 16"):
        ops.paged_kv_attention(q, kv, table, lens, mass=torch.zeros(table.shape))


def test_attention_refuses_too_many_requests_and_tokens():
    q, kv, table, lens = make(0, [5], 16, 4, 2, 64, torch.bfloat16)
    with pytest.raises(ValueError, match="at most"):
        ops.paged_kv_attention(q.expand(9000, -1, -1), kv, table.expand(9000, -1), lens.expand(9000))
    with pytest.raises(ValueError, match="too wide"):
        ops.paged_kv_attention(q, kv, table[:, :1].expand(1, 2**27), lens)
    with pytest.raises(ValueError, match="too large"):
        ops.paged_kv_attention(q.expand(64, -1, -1), kv, table[:, :1].expand(64, 2**26 - 1), lens.expand(64))
    q, kv, table, lens = make(0, [5], 1, 4, 2, 64, torch.bfloat16)
    with pytest.raises(ValueError, match="too large"):  # 2**31 blocks of one token
        ops.paged_kv_bounds(kv, table[:, :1].expand(4, 2**29), lens.repeat(4), torch.zeros(kv.shape[1], 2, 2, 64, dtype=kv.dtype))
    with pytest.raises(ValueError, match="a block"):
        ops.paged_kv_evict(torch.zeros(table.shape), table, lens, 4, block_size=65537)


def test_bounds_refuses(good):
    kv, table, lens = good["kv"], good["block_table"], good["context_lens"]
    ok = torch.zeros(kv.shape[1], 2, 2, 64, dtype=kv.dtype)
    for bounds, why in ((ok.float(), "bounds must"), (ok[:-1], "bounds must"), (wide(ok), "bounds must"),
                        (kv.flatten()[: ok.numel()].view(ok.shape), "overlap")):
        with pytest.raises(ValueError, match=why):
            ops.paged_kv_bounds(kv, table, lens, bounds)
    for new in (-1, 1.0, True, 2**31):
        with pytest.raises(ValueError, match="new_tokens"):
            ops.paged_kv_bounds(kv, table, lens, ok, new_tokens=new)
    with pytest.raises(ValueError, match="CUDA device"):
        ops.paged_kv_bounds(kv, table, lens, ok)


def test_select_refuses(good):
    q, table, lens = good["q"], good["block_table"], good["context_lens"]
    bounds = torch.zeros(6, 2, 2, 64, dtype=q.dtype)

    def call(q=q, bounds=bounds, keep=4, block_size=16, **more):
        return ops.paged_kv_select(q, bounds, table, lens, keep, block_size=block_size, **more)

    for change, why in ((dict(keep=0), "keep"), (dict(keep=2, sink=2, recent=1), "at least sink"), (dict(sink=-1), "sink"),
                        (dict(recent=-1), "recent"), (dict(block_size=0), "block_size"), (dict(q=q.half()), "q must be"),
                        (dict(bounds=bounds.float()), "bf16 or fp16"), (dict(bounds=bounds[:, :, :1]), "bounds must"),
                        (dict(bounds=bounds[..., :32]), "bounds must"), ({}, "CUDA device")):
        with pytest.raises(ValueError, match=why):
            call(**change)


def test_evict_refuses(good):
    table, lens = good["block_table"], good["context_lens"]
    mass = torch.zeros(table.shape)

    def call(mass=mass, budget=3, block_size=16, **more):
        return ops.paged_kv_evict(mass, table, lens, budget, block_size=block_size, **more)

    for change, why in ((dict(mass=mass.half()), "mass must"), (dict(mass=mass[:, :1]), "mass must"),
                        (dict(mass=wide(mass)), "contiguous"), (dict(budget=0), "budget"), (dict(recent=0), "recent"),
                        (dict(budget=2, sink=2), "at least sink"), (dict(block_size=0), "block_size"), ({}, "CUDA device")):
        with pytest.raises(ValueError, match=why):
            call(**change)


def test_a_query_that_splits_pairs_is_copied(good):
    from pcie_pool_b200._native import native_kv

    q = good["q"]
    odd = torch.zeros(q.numel() + 1, dtype=q.dtype)[1:].view(q.shape).copy_(q)
    spread = torch.zeros(*q.shape, 2, dtype=q.dtype)[..., 0].copy_(q)
    rows = torch.zeros(2, 8, 65, dtype=q.dtype)[..., :64].copy_(q)
    for x in (odd, spread, rows):
        got = native_kv().whole_pairs(x)
        assert got.data_ptr() % 4 == 0 and got.is_contiguous() and torch.equal(got, q)
    assert native_kv().whole_pairs(q).data_ptr() == q.data_ptr()


def test_offloader_saves_what_leaves(monkeypatch):
    from pcie_pool_b200.adapters.kv_offload import EvictedKV, _EvictsKV

    table = torch.tensor([[7, 3, 9, 4], [5, 6, -1, -1], [1, 2, 8, 0]], dtype=torch.int32)
    gone = [[3, 9, -1, -1], [-1] * 4, [2, -1, -1, -1]]
    at = [[1, 2, -1, -1], [-1] * 4, [1, -1, -1, -1]]
    asked = {}

    def evict(mass, block_table, context_lens, budget, **more):
        asked.update(more, budget=budget)
        t = [torch.tensor(x, dtype=torch.int32) for x in (gone, at, [2, 0, 1])]
        return ops.KVEviction(table, None, None, *t)

    monkeypatch.setattr(ops, "paged_kv_evict", evict)

    class Store(_EvictsKV):
        calls = []

        def save(self, ids, *host, host_off=0):
            self.calls.append((ids, host, host_off))
            return len(ids)

        def prefix_bytes(self, n):
            return 100 * n

    e, out = Store().evict(None, table, None, 3, "ptr", 4000, block_size=16, host_off=50, recent=2)
    assert asked == dict(budget=3, block_size=16, sink=1, recent=2)
    assert Store.calls == [([3, 9], ("ptr", 4000), 50), ([2], ("ptr", 4000), 250)]
    assert out == [EvictedKV(0, [3, 9], [1, 2], 50, 2), EvictedKV(2, [2], [1], 250, 1)]
