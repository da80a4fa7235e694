"""GPU tests of the paged-KV operators at the edges of what they take: entries that are no page, counts near their
limits, weights far below the leading one, values that are not finite, memory that arguments share."""

import math

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from pcie_pool_b200 import ops  # noqa: E402
from tests.paged_kv_cases import attention, best, make  # noqa: E402

BF16, FP16 = torch.bfloat16, torch.float16


# ---- eviction: entries that are no page of the cache -----------------------------------------------------


@pytest.mark.parametrize("n", [13, 700, 9000])
def test_evict_drops_entries_that_are_no_page(need_gpu, n):
    """They take no place in the budget, though they hold the most mass or stand first or last."""
    pages, budget = 2 * n, n // 2
    g = torch.Generator().manual_seed(n)
    table = torch.randperm(pages, generator=g)[:n].to(torch.int32)[None]
    mass = torch.rand(1, n, generator=g)
    bad = torch.tensor([0, 3, 4, n - 1])
    table[0, bad] = torch.tensor([pages, 2**31 - 1, -1, pages + 7], dtype=torch.int32)
    mass[0, bad] = 100.0
    can = [0 <= int(p) < pages for p in table[0]]
    stay = best(mass[0].tolist(), can, budget, 2, 3)
    gone = [j for j in range(n) if can[j] and j not in set(stay)]
    e = ops.paged_kv_evict(mass.cuda(), table.cuda(), torch.tensor([16 * n - 5], dtype=torch.int32).cuda(), budget,
                           block_size=16, sink=2, recent=3, pages=pages)
    assert e.block_table[0].tolist() == table[0, stay].tolist() + [-1] * (n - len(stay))
    assert e.evicted_blocks[0].tolist() == table[0, gone].tolist() + [-1] * (n - len(gone))
    assert e.evicted_index[0].tolist() == gone + [-1] * (n - len(gone))
    assert e.evicted_count.tolist() == [len(gone)] and e.context_lens.tolist() == [16 * len(stay)]


def test_offloader_evicts_around_entries_that_are_no_page(need_gpu):
    """A table with an entry past the cache: what is saved is the evicted pages' own, read back from the host."""
    from pcie_pool_b200.adapters import PagedKVOffloader
    from pcie_pool_b200.parallel.engine import PoolEngine
    from pcie_pool_b200.utils.host_memory import PinnedHostBuffer

    pages = 24
    g = torch.Generator().manual_seed(1)
    kv = torch.randn(2, pages, 16, 2, 64, generator=g).to(BF16).cuda()
    table = torch.randperm(pages, generator=g)[:12].to(torch.int32)[None]
    table[0, 2], table[0, 5] = pages, pages + 1000
    mass = torch.rand(1, 12, generator=g)
    mass[0, [2, 5]] = 50.0
    host = PinnedHostBuffer(1 << 20)
    try:
        store = PagedKVOffloader(PoolEngine([0], slot_bytes=1 << 20, slots=3, timeout_s=10.0), [kv], target=0)
        e, gone = store.evict(mass.cuda(), table.cuda(), torch.tensor([12 * 16], dtype=torch.int32).cuda(), 4, host.ptr, 1 << 20,
                              block_size=16)
        assert len(gone) == 1 and len(gone[0].blocks) == 6 and all(0 <= p < pages for p in gone[0].blocks)
        assert set(e.block_table[0, :4].tolist()) | set(gone[0].blocks) == {int(p) for p in table[0] if p < pages}
        saved = kv[:, gone[0].blocks].clone()
        kv.zero_()
        store.restore(gone[0].blocks, host.ptr, 1 << 20, host_off=gone[0].host_off)
        torch.cuda.synchronize()
        assert torch.equal(kv[:, gone[0].blocks], saved)
    finally:
        host.release()


# ---- selection ----------------------------------------------------------------------------------------


def test_select_of_the_most_blocks_there_can_be(need_gpu):
    """keep = 2**31 - 1: the places behind the row are filled to the last, and nothing before the row."""
    if torch.cuda.mem_get_info()[0] < 16 << 30:
        pytest.skip("needs 16 GB")
    q, kv, table, lens = make(70, [40], 16, 2, 1, 8, BF16)
    bounds = torch.zeros(kv.shape[1], 1, 2, 8, dtype=BF16, device="cuda")
    out = ops.paged_kv_select(q.cuda(), bounds, table.cuda(), lens.cuda(), 2**31 - 1, block_size=16)
    assert out.shape == (1, 1, 2**31 - 1) and out[0, 0, :3].tolist() == [0, 1, 2]
    assert all((part == -1).all() for part in out[0, 0, 3:].split(1 << 28))


# ---- weights far below the leading one --------------------------------------------------------------------


def check_attention(q, kv, table, lens, out, lse, **more):
    from tests.test_gpu_paged_kv import check_attention as check

    return check(q, kv, table, lens, out, lse, **more)


def with_a_leading_token(dtype, heads, kv_heads, dim, tokens, gap, where, seed):
    """One token `gap` nats above the others, with values a thousand times smaller: what the others give is the result."""
    q, kv, table, lens = make(seed, [tokens], 16, heads, kv_heads, dim, dtype)
    q[..., 0], q[..., 1:] = 1.0, 0.0
    kv[0, ..., 0] = kv[0, ..., 0].abs().clamp(max=0.5)
    at = (table[0, where // 16], where % 16)
    kv[0][at][:, 0] = gap
    kv[1] = kv[1].abs() + 0.5
    kv[1][at] = kv[1][at] / 1024
    return q, kv, table, lens


@pytest.mark.parametrize("gap", [8.0, 12.0, 14.0, 16.0, 18.0, 20.0])
@pytest.mark.parametrize("heads,kv_heads,dim,tokens,where", [
    (600, 600, 8, 800, 0), (600, 600, 8, 800, 400), (5400, 600, 8, 320, 0),  # a range holds all tokens; heads alone, and nine to a key head
    (300, 300, 256, 320, 7),
    (4, 1, 64, 800, 3), (18, 1, 128, 800, 3)])                               # many ranges, joined
def test_small_weights_are_not_lost_beside_a_leading_one(need_gpu, heads, kv_heads, dim, tokens, where, gap):
    q, kv, table, lens = with_a_leading_token(FP16, heads, kv_heads, dim, tokens, gap, where, 71)
    out, lse = ops.paged_kv_attention(q.cuda(), kv.cuda(), table.cuda(), lens.cuda(), scale=1.0, return_lse=True)
    check_attention(q, kv, table, lens, out, lse, scale=1.0)


@pytest.mark.parametrize("gap", [8.0, 40.0, 80.0])
def test_small_weights_in_bf16(need_gpu, gap):
    q, kv, table, lens = with_a_leading_token(BF16, 600, 600, 8, 800, gap, 400, 72)
    out, lse = ops.paged_kv_attention(q.cuda(), kv.cuda(), table.cuda(), lens.cuda(), scale=1.0, return_lse=True)
    check_attention(q, kv, table, lens, out, lse, scale=1.0)


@pytest.mark.parametrize("heads,kv_heads", [(600, 600), (5400, 600)])
def test_large_values_in_fp16(need_gpu, heads, kv_heads):
    """Values at the type's end: what is summed is larger than they are by the weights' scale and the tokens' number."""
    q, kv, table, lens = make(73, [320], 16, heads, kv_heads, 8, FP16)
    kv[1] = torch.where(kv[1] > 0, 65504.0, -65504.0).to(FP16).where(~torch.isnan(kv[1]), kv[1])
    kv[1][..., 0] = kv[1][..., 0].abs()
    out, lse = ops.paged_kv_attention(q.cuda(), kv.cuda(), table.cuda(), lens.cuda(), scale=0.25, return_lse=True)
    check_attention(q, kv, table, lens, out, lse, scale=0.25)


# ---- what is written, and autograd -------------------------------------------------------------------------


def test_what_is_written_is_known_to_autograd(need_gpu):
    q, kv, table, lens = (t.cuda() for t in make(74, [40, 5], 16, 8, 2, 64, BF16))
    w = torch.ones(q.shape, dtype=BF16, device="cuda", requires_grad=True)
    m = torch.ones(table.shape, device="cuda", requires_grad=True)
    b = torch.ones(kv.shape[1], 2, 2, 64, dtype=BF16, device="cuda", requires_grad=True)
    out, mass, bounds = torch.zeros_like(q), torch.zeros(table.shape, device="cuda"), torch.zeros_like(b, requires_grad=False)
    graphs = [(w * out).sum(), (m * mass).sum(), (b * bounds).sum()]  # each saves what is written below
    ops.paged_kv_attention(q, kv, table, lens, out=out, mass=mass)
    ops.paged_kv_bounds(kv, table, lens, bounds)
    assert out._version == 1 and mass._version == 1 and bounds._version == 1
    for loss in graphs:
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()
    with torch.inference_mode():  # tensors that have no versions
        out = torch.zeros_like(q)
        ops.paged_kv_attention(q, kv, table, lens, out=out)
        assert out.abs().sum() > 0


# ---- layouts ---------------------------------------------------------------------------------------------


@pytest.mark.parametrize("dim,lens,block,kv_heads", [(1, [9], 16, 2), (2, [3, 4], 1, 2), (3, [70, 5], 16, 1)])
def test_any_stride_of_a_dimension_of_one(need_gpu, dim, lens, block, kv_heads):
    q, kv, table, lens = make(75, lens, block, 2 * kv_heads, kv_heads, 64, BF16, pages_extra=0)
    assert kv.shape[dim] == 1
    strides = list(kv.stride())
    strides[dim] = 3
    odd = kv.cuda().as_strided(kv.shape, strides)
    out, lse = ops.paged_kv_attention(q.cuda(), odd, table.cuda(), lens.cuda(), return_lse=True)
    check_attention(q, kv, table, lens, out, lse)
    bounds = [torch.zeros(kv.shape[1], kv_heads, 2, 64, dtype=BF16, device="cuda") for _ in range(2)]
    for k, b in zip((odd, kv.cuda()), bounds):
        ops.paged_kv_bounds(k, table.cuda(), lens.cuda(), b)
    assert torch.equal(*bounds)


# ---- scores -----------------------------------------------------------------------------------------------


@pytest.mark.parametrize("other", ["nothing", "nan", "inf"])
@pytest.mark.parametrize("dim", [8, 256])
def test_a_score_does_not_hang_on_its_neighbours(need_gpu, other, dim):
    """Block 1 is 1 + 2^-24 and two numbers that 64 bits round away one by one, but not when they are added first: it would
    then round to more than the 1 of block 0.  A neighbour that is not finite must not change how it is summed."""
    bounds = torch.zeros(9, 1, 2, dim, dtype=BF16)
    bounds[0, 0, 1, 0] = 1.0
    bounds[1, 0, 1, :2] = torch.tensor([1.0, 2.0 ** -24])
    bounds[1, 0, 0, 2:4] = -3 * 2.0 ** -55
    if other != "nothing":
        bounds[2, 0, :, 0] = -math.inf if other == "inf" else math.nan
    q = torch.zeros(1, 1, dim, dtype=BF16)
    q[0, 0, :4] = torch.tensor([1.0, 1.0, -1.0, -1.0])
    table, lens = torch.arange(9, dtype=torch.int32)[None].cuda(), torch.tensor([9], dtype=torch.int32).cuda()
    got = ops.paged_kv_select(q.cuda(), bounds.cuda(), table, lens, 1, block_size=1, sink=0, recent=0)
    assert got.tolist() == [[[0]]]


@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_a_channel_without_a_query_adds_nothing_to_a_score(need_gpu, dtype):
    bounds = torch.zeros(5, 1, 2, 8, dtype=dtype)
    bounds[0, 0, 1, 0] = 1.0
    bounds[1, 0, 1, 0], bounds[1, 0, 1, 3], bounds[1, 0, 0, 4] = 2.0, math.inf, math.nan   # channels 3 and 4 have no query
    bounds[2, 0, 0, 0], bounds[2, 0, 1, 0] = math.nan, 3.0
    bounds[3, 0, 0, 0], bounds[3, 0, 1, 0] = 4.0, math.nan
    bounds[4, 0, :, 0] = math.nan
    q = torch.zeros(1, 2, 8, dtype=dtype)
    q[0, :, 0] = torch.tensor([1.0, 0.0])
    table, lens = torch.arange(5, dtype=torch.int32)[None].cuda(), torch.tensor([5], dtype=torch.int32).cuda()
    for keep, want in enumerate(([3], [2, 3], [1, 2, 3], [0, 1, 2, 3], [0, 1, 2, 3, 4]), 1):
        got = ops.paged_kv_select(q.cuda(), bounds.cuda(), table, lens, keep, block_size=1, sink=0, recent=0)
        assert got[0, 0].tolist() == want


# ---- what is not finite --------------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("heads", [4, 24])
@pytest.mark.parametrize("tokens", [40, 3000])
def test_what_is_not_finite_shows_where_it_counts(need_gpu, dtype, heads, tokens):
    q, kv, table, lens = make(76, [tokens] * 4, 16, heads, 2, 64, dtype)
    G = heads // 2
    q[:, :, 0] = q[:, :, 0].abs() + 0.5
    kv[1, table[0, 1], 3, 1, 5] = math.inf       # a value: channel 5 of the second key head's queries
    kv[1, table[1, 1], 3, 0, 6] = -math.inf
    kv[0, table[2, 0], 7, 1, 0] = math.inf       # a key: scores of plus infinity
    kv[0, table[3, 0], 7, 0, 0] = -math.inf      # of minus infinity, whose value does not matter
    kv[1, table[3, 0], 7, 0] = 0.0
    mass = torch.zeros(table.shape, device="cuda")
    out, lse = ops.paged_kv_attention(q.cuda(), kv.cuda(), table.cuda(), lens.cuda(), mass=mass, return_lse=True)
    bad = ~torch.isfinite(out).cpu()
    want = torch.zeros_like(bad)
    want[0, G:, 5] = want[1, :G, 6] = want[2, G:] = True
    assert torch.equal(bad, want)
    assert torch.isnan(out[2, G:]).all() and torch.isnan(lse[2, G:]).all()
    assert torch.isfinite(lse[:2]).all() and torch.isfinite(lse[2, :G]).all() and torch.isfinite(lse[3]).all()
    n = -(-tokens // 16)
    assert torch.isfinite(mass[[0, 1, 3]]).all() and torch.isnan(mass[2, :n]).all() and (mass[2, n:] == 0).all()
    # the first key head's token of minus infinity as if it were not there: the last one in its place
    page, at = table[3, (tokens - 1) // 16], (tokens - 1) % 16
    without = kv.clone()
    without[:, table[3, 0], 7, 0] = kv[:, page, at, 0]
    for rows, cache, length in ((slice(0, G), without, tokens - 1), (slice(G, heads), kv, tokens)):
        ref, _, _, err, _ = attention(q[3:], cache, table[3:], torch.tensor([length]))
        tol = err + torch.finfo(dtype).eps / 2 * (ref.abs() + err) + (2.0 ** -25 if dtype == FP16 else 0.0)
        assert ((out[3:].cpu().double() - ref).abs() <= tol)[:, rows].all()


# ---- the largest numbers of requests and tokens a page ------------------------------------------------------------


def test_mass_of_more_requests_than_ranges(need_gpu):
    lens = [(i * 37) % 90 for i in range(700)]
    q, kv, table, lens = make(77, lens, 16, 4, 2, 64, FP16)
    mass = torch.zeros(table.shape, device="cuda")
    out, lse = ops.paged_kv_attention(q.cuda(), kv.cuda(), table.cuda(), lens.cuda(), mass=mass, return_lse=True)
    weight, lse_err = check_attention(q, kv, table, lens, out, lse)
    tol = weight * (3 * lse_err.amax(1, keepdim=True) + 84 * 2.0 ** -24 + 2.0 ** -20) + 2.0 ** -24 * weight
    assert ((mass.cpu().double() - weight).abs() <= tol).all()


@pytest.mark.parametrize("dim,dtype", [(64, BF16), (128, FP16), (256, BF16)])
def test_the_most_requests(need_gpu, dim, dtype):
    """4096 requests of 0 to 6 tokens, two of them long: attention, bounds, selection and eviction."""
    from tests.paged_kv_cases import scores

    lens = [i % 7 for i in range(4096)]
    lens[1000], lens[4095] = 500, 333
    q, kv, table, lens = make(78, lens, 16, 2, 1, dim, dtype)
    qg, kg, tg, lg = (t.cuda() for t in (q, kv, table, lens))
    mass = torch.zeros(table.shape, device="cuda")
    out, lse = ops.paged_kv_attention(qg, kg, tg, lg, mass=mass, return_lse=True)
    weight, _ = check_attention(q, kv, table, lens, out, lse)
    assert ((mass.cpu().double() - weight).abs() <= 1e-4 * weight + 1e-6).all()
    bounds = torch.zeros(kv.shape[1], 1, 2, dim, dtype=dtype)
    for b in range(4096):
        for j in range(-(-int(lens[b]) // 16)):
            k = kv[0, table[b, j], : min(16, int(lens[b]) - 16 * j)]
            bounds[table[b, j]] = torch.stack((k.amin(0), k.amax(0)), 1)
    got = ops.paged_kv_bounds(kg, tg, lg, torch.zeros_like(bounds).cuda())
    assert torch.equal(got.cpu(), bounds)
    blocks = ops.paged_kv_select(qg, got, tg, lg, 3, block_size=16).cpu()
    e = ops.paged_kv_evict(mass, tg, lg, 3, block_size=16)
    m = mass.cpu()
    for b in (0, 1, 6, 1000, 2047, 4094, 4095):
        n = -(-int(lens[b]) // 16)
        at = best(scores(q[b], bounds, [int(p) for p in table[b, :n]])[0].tolist() if n else [], [True] * n, 3, 1, 1)
        assert blocks[b, 0].tolist() == at + [-1] * (3 - len(at))
        stay = best(m[b, :n].tolist(), [True] * n, 3, 1, 1)
        assert e.block_table[b, : len(stay)].tolist() == table[b, stay].tolist() and int(e.evicted_count[b]) == n - len(stay)
    assert (blocks[:, 0, 0].ge(0) == lens.gt(0)).all() and (e.evicted_count.cpu() == (-(-lens // 16) - 3).clamp(min=0)).all()


@pytest.mark.parametrize("block", [65536, 4099])
def test_the_largest_pages(need_gpu, block):
    q, kv, table, lens = make(79, [70000, 5, 65537], block, 2, 1, 8, BF16, pages_extra=0, width_extra=0)
    out, lse = ops.paged_kv_attention(q.cuda(), kv.cuda(), table.cuda(), lens.cuda(), return_lse=True)
    check_attention(q, kv, table, lens, out, lse)
    got = ops.paged_kv_bounds(kv.cuda(), table.cuda(), lens.cuda(), torch.zeros(kv.shape[1], 1, 2, 8, dtype=BF16, device="cuda")).cpu()
    for b, n in enumerate(lens.tolist()):
        for j in range(-(-n // block)):
            k = kv[0, table[b, j], : min(block, n - j * block)]
            assert torch.equal(got[table[b, j]], torch.stack((k.amin(0), k.amax(0)), 1))


# ---- the same block and page again ---------------------------------------------------------------------------------


@pytest.mark.parametrize("heads", [4, 24])
def test_the_same_block_and_page_again(need_gpu, heads):
    """A block listed twice counts twice, a page in two places of a table or in two requests is read in each; of a list only as
    many entries count as the request has blocks."""
    q, kv, table, lens = make(80, [75, 75, 33], 16, heads, 2, 64, BF16)
    table[0, 3] = table[0, 1]
    table[1] = table[0]
    out, lse = ops.paged_kv_attention(q.cuda(), kv.cuda(), table.cuda(), lens.cuda(), return_lse=True)
    check_attention(q, kv, table, lens, out, lse)
    blocks = torch.tensor([[[2, 2, 0, 4, 4, 1, 3], [4, 0, 0, 0, 0, 0, 0]], [[1, 3, 1, 3, 0, 2, 2], [0, 1, 2, 3, 4, 0, 1]],
                           [[2, 2, 2, 0, 1, 0, 1], [1, -1, 1, 2, 2, 2, 2]]], dtype=torch.int32)
    out, lse = ops.paged_kv_attention(q.cuda(), kv.cuda(), table.cuda(), lens.cuda(), blocks=blocks.cuda(), return_lse=True)
    check_attention(q, kv, table, lens, out, lse, blocks=blocks)
