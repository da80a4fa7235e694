"""GPU tests of the paged-KV operators against 64-bit oracles (tests/paged_kv_cases.py)."""

import math

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from pcie_pool_b200 import ops  # noqa: E402
from tests.paged_kv_cases import attention, best, make, scores, to_gpu  # noqa: E402

BF16, FP16 = torch.bfloat16, torch.float16


def check_attention(q, kv, table, lens, out, lse, **more):
    ref, ref_lse, weight, err, lse_err = attention(q, kv, table, lens, **more)
    got = out.cpu().double()
    # the result's own rounding, half a step of its type, and fp16's smallest step
    tol = err + torch.finfo(q.dtype).eps / 2 * (ref.abs() + err) + (2.0 ** -25 if q.dtype == FP16 else 0.0)
    assert torch.equal(torch.isnan(got), torch.isnan(ref))
    bad = (got - ref).abs() > tol
    assert not bad.any(), ((got - ref).abs() / tol).max()
    got = lse.cpu().double()
    assert torch.equal(got == -math.inf, ref_lse == -math.inf)
    some = ref_lse > -math.inf
    assert ((got - ref_lse).abs()[some] <= lse_err[some]).all()
    return weight, lse_err


def run_attention(q, kv, table, lens, blocks=None, scale=None):
    out, lse = ops.paged_kv_attention(q.cuda(), to_gpu(kv), table.cuda(), lens.cuda(), scale=scale, return_lse=True,
                                      blocks=None if blocks is None else blocks.cuda())
    return check_attention(q, kv, table, lens, out, lse, blocks=blocks, scale=scale)


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("dim", [8, 64, 80, 128, 192, 256])
@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (4, 4), (10, 2), (8, 1), (18, 2), (40, 1)])
def test_attention_shapes(need_gpu, dtype, dim, heads, kv_heads):
    run_attention(*make(dim + heads, [1, 33, 0, 147], 16, heads, kv_heads, dim, dtype))


@pytest.mark.parametrize("block", [1, 3, 8, 16, 24, 32, 100, 256])
def test_attention_block_sizes(need_gpu, block):
    run_attention(*make(block, [1, 15, 16, 17, 0, 255, 256, 257, 31], block, 8, 2, 64, BF16))


@pytest.mark.parametrize("layout", ["planes", "pages", "heads", "padded"])
def test_attention_cache_layouts(need_gpu, layout):
    run_attention(*make(5, [70, 0, 3, 129], 16, 6, 3, 128, FP16, layout=layout))


def test_attention_long_and_short_together(need_gpu):
    run_attention(*make(7, [1, 9000, 2, 0, 0, 17, 1, 2500, 16, 1], 16, 4, 2, 64, BF16))


def test_attention_many_short_requests(need_gpu):
    run_attention(*make(8, [(i * 7) % 40 for i in range(700)], 16, 4, 2, 64, FP16))


def test_attention_all_empty(need_gpu):
    q, kv, table, lens = make(9, [0, 0, 0], 16, 4, 2, 64, BF16)
    out, lse = ops.paged_kv_attention(q.cuda(), kv.cuda(), table.cuda(), lens.cuda(), return_lse=True)
    assert (out == 0).all() and (lse == -math.inf).all()
    none = ops.paged_kv_attention(q[:0].cuda(), kv.cuda(), table[:0].cuda(), lens[:0].cuda())
    assert none.shape == (0, 4, 64)
    no_pages = ops.paged_kv_attention(q.cuda(), kv[:, :0].cuda(), table[:, :0].cuda(), lens.cuda() + 5)
    assert (no_pages == 0).all()


def test_attention_leaves_out_blocks_that_are_not_resident(need_gpu):
    q, kv, table, lens = make(10, [100, 64, 40, 16], 16, 8, 2, 64, BF16)
    table[0, 1], table[0, 6] = -1, -7
    table[1, 0], table[1, 3] = kv.shape[1], 2**31 - 1
    table[2, :] = -1
    run_attention(q, kv, table, lens)


def test_attention_cuts_lengths_to_the_table(need_gpu):
    q, kv, table, lens = make(11, [64, 64, 64], 16, 8, 2, 64, BF16, width_extra=0)
    run_attention(q, kv, table, torch.tensor([2**31 - 1, 65, -3], dtype=torch.int32))


def test_attention_large_scores(need_gpu):
    # one key far above the others, and scores that exp() of would not hold
    q, kv, table, lens = make(12, [300, 50], 16, 8, 2, 64, BF16)
    run_attention(q, kv, table, lens, scale=40.0)
    run_attention(q, kv, table, lens, scale=0.0)
    run_attention(q, kv, table, lens, scale=-0.5)


def test_attention_keeps_nan_of_a_token_that_counts(need_gpu):
    q, kv, table, lens = make(13, [40, 40], 16, 4, 2, 64, BF16)
    kv[1, table[0, 1], 3, 1, 5] = math.nan
    kv[0, table[1, 0], 0, 0, 0] = math.nan
    out, lse = ops.paged_kv_attention(q.cuda(), kv.cuda(), table.cuda(), lens.cuda(), return_lse=True)
    nan = torch.isnan(out).cpu()
    assert nan[0, 2:, 5].all() and nan[0].sum() == 2
    assert nan[1, :2].all() and not nan[1, 2:].any()
    assert torch.isnan(lse[1, :2]).all() and not torch.isnan(lse[0]).any()


def test_attention_rows_of_minus_infinity(need_gpu):
    # keys whose every score is -inf count for nothing; next to finite ones they leave those as they are
    q, kv, table, lens = make(14, [40, 33], 16, 4, 2, 64, BF16)
    q = q.abs()
    kv[0, table[0, 0], 2] = -math.inf
    for j in range(3):
        kv[0, table[1, j], : min(16, 33 - 16 * j), 0] = -math.inf
    out, lse = ops.paged_kv_attention(q.cuda(), kv.cuda(), table.cuda(), lens.cuda(), return_lse=True)
    assert (out[1, :2] == 0).all() and (lse[1, :2] == -math.inf).all()
    assert torch.isfinite(out).all() and torch.isfinite(lse[0]).all() and torch.isfinite(lse[1, 2:]).all()


def test_attention_views_of_wider_tensors(need_gpu):
    q, kv, table, lens = make(15, [70, 5, 33], 16, 8, 2, 64, BF16)
    fused = torch.zeros(3, 8 + 4, 64, dtype=BF16, device="cuda")
    fused[:, :8] = q.cuda()
    odd = torch.zeros(3 * 8 * 64 + 1, dtype=BF16, device="cuda")[1:].view(3, 8, 64).copy_(q)
    spread = torch.zeros(3, 8, 64, 2, dtype=BF16, device="cuda")[..., 0].copy_(q)
    big = torch.zeros(3, table.shape[1] + 9, dtype=torch.int32, device="cuda")
    big[:, 2: 2 + table.shape[1]] = table.cuda()
    view = big[:, 2: 2 + table.shape[1]]
    kvg = kv.cuda()
    for x in (fused[:, :8], odd, spread):
        out, lse = ops.paged_kv_attention(x, kvg, view, lens.cuda(), return_lse=True)
        check_attention(q, kv, table, lens, out, lse)


def test_attention_writes_to_out_and_nowhere_else(need_gpu):
    q, kv, table, lens = make(16, [70, 5, 0], 16, 8, 2, 64, BF16)
    buf = torch.full((5, 8, 64), 7.0, dtype=BF16, device="cuda")
    out = ops.paged_kv_attention(q.cuda(), kv.cuda(), table.cuda(), lens.cuda(), out=buf[1:4])
    assert out.data_ptr() == buf[1:4].data_ptr()
    assert (buf[0] == 7).all() and (buf[4] == 7).all()
    ref = ops.paged_kv_attention(q.cuda(), kv.cuda(), table.cuda(), lens.cuda())
    assert torch.equal(out, ref)


def test_attention_is_the_same_every_time(need_gpu):
    q, kv, table, lens = (t.cuda() for t in make(17, [5000, 77, 1200, 16], 16, 16, 4, 128, BF16))
    mass = torch.zeros(table.shape, device="cuda")
    first = ops.paged_kv_attention(q, kv, table, lens, mass=mass, return_lse=True)
    for _ in range(5):
        again = torch.zeros_like(mass)
        got = ops.paged_kv_attention(q, kv, table, lens, mass=again, return_lse=True)
        assert torch.equal(got[0], first[0]) and torch.equal(got[1], first[1]) and torch.equal(again, mass)


def test_attention_offsets_past_32_bits(need_gpu):
    pages = 150_000
    kv = torch.zeros(2, pages, 16, 8, 128, dtype=BF16, device="cuda")  # 2.4e9 values a plane
    q, small, table, lens = make(18, [90, 40], 16, 16, 8, 128, BF16, pages_extra=0)
    far = torch.arange(small.shape[1]) * 7 + pages - 7 * small.shape[1]
    kv[:, far.cuda()] = small.cuda()
    out, lse = ops.paged_kv_attention(q.cuda(), kv, far.to(torch.int32)[table.long()].cuda(), lens.cuda(), return_lse=True)
    check_attention(q, small, table, lens, out, lse)


@pytest.mark.parametrize("heads,kv_heads,dim,block,dtype", [(8, 2, 64, 16, BF16), (5, 5, 128, 32, FP16), (24, 2, 128, 48, BF16),
                                                            (33, 1, 64, 128, FP16)])
def test_mass(need_gpu, heads, kv_heads, dim, block, dtype):
    lens = [1, 400, 0, 129, 48, 47]
    q, kv, table, lens = make(dim + block, lens, block, heads, kv_heads, dim, dtype)
    table[1, 1] = -1
    wide = torch.rand(len(lens), table.shape[1] + 5, device="cuda")
    before = wide.clone()
    mass = wide[:, 2: 2 + table.shape[1]]
    out, lse = ops.paged_kv_attention(q.cuda(), kv.cuda(), table.cuda(), lens.cuda(), mass=mass, return_lse=True)
    weight, lse_err = check_attention(q, kv, table, lens, out, lse)
    old = before[:, 2: 2 + table.shape[1]].cpu().double()
    got = mass.cpu().double()
    # each head's weight is off by what its scores and its sum are, and by the log and exp of a tile's sum; then heads add up
    tol = weight * (3 * lse_err.amax(1, keepdim=True) + (heads + 80) * 2.0 ** -24 + 2.0 ** -20) + 2.0 ** -24 * (old + weight)
    assert ((got - (old + weight)).abs() <= tol).all()
    for b in range(len(lens)):  # behind the request's blocks nothing is touched
        n = -(-int(lens[b]) // block)
        assert torch.equal(mass[b, n:].cpu(), before[b, 2 + n: 2 + table.shape[1]].cpu())
    assert torch.equal(wide[:, :2], before[:, :2]) and torch.equal(wide[:, -3:], before[:, -3:])


@pytest.mark.parametrize("block", [16, 8, 40])
def test_sparse_attention_reads_the_listed_blocks(need_gpu, block):
    q, kv, table, lens = make(20, [333, 16, 0, 1000], block, 12, 3, 64, BF16)
    g = torch.Generator().manual_seed(1)
    blocks = torch.full((4, 3, 9), -1, dtype=torch.int32)
    for b in range(4):
        n = -(-int(lens[b]) // block)
        for h in range(3):
            m = min(9, n)
            blocks[b, h, :m] = torch.randperm(n, generator=g)[:m].to(torch.int32)
    blocks[3, 1, 4] = -1                  # no block
    blocks[3, 2, 0] = 2**31 - 1           # not of this request
    blocks[0, 0, 1] = -2**31
    table[3, int(blocks[3, 0, 2])] = -5   # listed but not resident
    run_attention(q, kv, table, lens, blocks=blocks)


def test_sparse_attention_of_no_blocks(need_gpu):
    q, kv, table, lens = (t.cuda() for t in make(21, [333, 16], 16, 4, 2, 64, BF16))
    for blocks in (torch.empty(2, 2, 0, dtype=torch.int32, device="cuda"), torch.full((2, 2, 3), -1, dtype=torch.int32, device="cuda")):
        out, lse = ops.paged_kv_attention(q, kv, table, lens, blocks=blocks, return_lse=True)
        assert (out == 0).all() and (lse == -math.inf).all()


@pytest.mark.parametrize("kv_heads,heads,dim", [(1300, 1300, 8), (300, 600, 256)])
def test_more_key_heads_than_warps(need_gpu, kv_heads, heads, dim):
    q, kv, table, lens = make(22, [40, 0, 17], 16, heads, kv_heads, dim, BF16)
    mass = torch.zeros(table.shape, device="cuda") if heads <= 1024 else None
    out, lse = ops.paged_kv_attention(q.cuda(), kv.cuda(), table.cuda(), lens.cuda(), mass=mass, return_lse=True)
    weight, lse_err = check_attention(q, kv, table, lens, out, lse)
    if mass is not None:
        tol = weight * (3 * lse_err.amax(1, keepdim=True) + (heads + 80) * 2.0 ** -24 + 2.0 ** -20)
        assert ((mass.cpu().double() - weight).abs() <= tol + 2.0 ** -24 * weight).all()


def test_nothing_to_do(need_gpu):
    q, kv, table, lens = (t.cuda() for t in make(23, [40, 17], 16, 4, 2, 64, BF16))
    bounds = torch.full((kv.shape[1], 2, 2, 64), 3.0, dtype=BF16, device="cuda")
    none, mass = table[:, :0], torch.zeros(2, 0, device="cuda")
    assert (ops.paged_kv_attention(q, kv, none, lens, mass=mass) == 0).all()
    assert (ops.paged_kv_bounds(kv, none, lens, bounds) == 3).all()
    assert (ops.paged_kv_select(q, bounds, none, lens, 4, block_size=16) == -1).all()
    e = ops.paged_kv_evict(mass, none, lens, 4, block_size=16)
    assert e.block_table.shape == (2, 0) and (e.context_lens == 0).all() and (e.evicted_count == 0).all()
    empty = table[:0], lens[:0]
    assert ops.paged_kv_select(q[:0], bounds, *empty, 4, block_size=16).shape == (0, 2, 4)
    assert (ops.paged_kv_bounds(kv, *empty, bounds) == 3).all()
    assert ops.paged_kv_evict(torch.zeros(0, table.shape[1], device="cuda"), *empty, 4, block_size=16).context_lens.shape == (0,)


# ---- bounds ---------------------------------------------------------------------------------


def plain_bounds(kv, table, lens, bounds, new):
    bs = kv.shape[2]
    for b in range(len(lens)):
        n = min(int(lens[b]), table.shape[1] * bs)
        for j in range(-(-n // bs) if n > 0 else 0):
            p = int(table[b, j])
            if not 0 <= p < kv.shape[1] or (new is not None and (j + 1) * bs <= n - new):
                continue
            k = kv[0, p, : min(bs, n - j * bs)]
            bounds[p] = torch.stack((k.amin(0), k.amax(0)), 1)
    return bounds


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("dim,kv_heads,block", [(8, 1, 16), (64, 3, 16), (128, 8, 16), (80, 2, 24), (256, 4, 1), (128, 40, 7), (64, 1, 130)])
@pytest.mark.parametrize("new", [None, 0, 1, 17, 100000])
def test_bounds(need_gpu, dtype, dim, kv_heads, block, new):
    q, kv, table, lens = make(dim + block, [1, 100, 0, 64, 65], block, kv_heads, kv_heads, dim, dtype)
    table[1, 0] = -1
    table[3, 1 % table.shape[1]] = kv.shape[1]
    start = torch.full((kv.shape[1], kv_heads, 2, dim), 9.0, dtype=dtype)
    if new == 0:
        ref = start.clone()
    else:
        ref = plain_bounds(kv, table, lens, start.clone(), new)
    got = start.cuda()
    assert ops.paged_kv_bounds(to_gpu(kv), table.cuda(), lens.cuda(), got, new_tokens=new) is got
    assert torch.equal(got.cpu(), ref)


@pytest.mark.parametrize("layout", ["pages", "heads", "padded"])
def test_bounds_cache_layouts(need_gpu, layout):
    q, kv, table, lens = make(3, [70, 16, 129], 16, 3, 3, 64, BF16, layout=layout)
    start = torch.zeros(kv.shape[1], 3, 2, 64, dtype=BF16)
    got = ops.paged_kv_bounds(to_gpu(kv), table.cuda(), lens.cuda(), start.cuda())
    assert torch.equal(got.cpu(), plain_bounds(kv, table, lens, start, None))


def test_bounds_pass_over_nan_and_keep_infinities(need_gpu):
    q, kv, table, lens = make(4, [20], 16, 1, 1, 8, BF16)
    kv[0, table[0, 0], 3, 0, 0] = math.nan
    kv[0, table[0, 0], 0, 0, 0] = math.nan
    kv[0, table[0, 0], 5, 0, 1] = math.inf
    kv[0, table[0, 0], 6, 0, 2] = -math.inf
    got = ops.paged_kv_bounds(kv.cuda(), table.cuda(), lens.cuda(), torch.zeros(kv.shape[1], 1, 2, 8, dtype=BF16, device="cuda"))
    k = kv[0, table[0, 0], :, 0]
    lo, hi = got[table[0, 0].item(), 0].cpu()
    assert lo[0] == k[:, 0].nan_to_num(99).min() and hi[0] == k[:, 0].nan_to_num(-99).max()
    assert hi[1] == math.inf and lo[2] == -math.inf


# ---- selection --------------------------------------------------------------------------------


def plain_select(q, bounds, table, lens, keep, block, sink, recent):
    Hk = bounds.shape[1]
    out = torch.full((len(lens), Hk, keep), -1, dtype=torch.int32)
    for b in range(len(lens)):
        n = max(0, min(-(-int(lens[b]) // block), table.shape[1]))
        can = [0 <= int(table[b, j]) < bounds.shape[0] for j in range(n)]
        sc = scores(q[b], bounds, [int(table[b, j]) if can[j] else 0 for j in range(n)])
        for h in range(Hk):
            at = best(sc[h].tolist(), can, keep, sink, recent)
            out[b, h, : len(at)] = torch.tensor(at, dtype=torch.int32)
    return out


@pytest.mark.parametrize("heads,kv_heads,dim,dtype", [(8, 2, 128, BF16), (3, 3, 64, FP16), (24, 1, 80, BF16), (32, 8, 128, FP16),
                                                      (16, 2, 256, BF16), (5, 1, 8, BF16)])
@pytest.mark.parametrize("keep,sink,recent", [(1, 0, 0), (1, 0, 1), (7, 1, 2), (64, 3, 5)])
def test_select(need_gpu, heads, kv_heads, dim, dtype, keep, sink, recent):
    q, kv, table, lens = make(dim + keep, [1, 0, 700, 90, 1601], 16, heads, kv_heads, dim, dtype)
    table[2, 3], table[2, 0], table[4, 9] = -1, kv.shape[1] + 5, -9
    bounds = plain_bounds(kv, table, lens, torch.full((kv.shape[1], kv_heads, 2, dim), math.nan, dtype=dtype), None)
    got = ops.paged_kv_select(q.cuda(), bounds.cuda(), table.cuda(), lens.cuda(), keep, block_size=16, sink=sink, recent=recent)
    assert torch.equal(got.cpu(), plain_select(q, bounds, table, lens, keep, 16, sink, recent))


@pytest.mark.parametrize("n", [511, 512, 513, 4096, 4097, 20000, 70001])
def test_select_many_blocks_with_ties(need_gpu, n):
    # scores from few values: most places of the border are ties
    g = torch.Generator().manual_seed(n)
    bounds = torch.randint(-2, 3, (50, 2, 2, 8), generator=g).to(BF16)
    table = torch.randint(0, 50, (2, n), generator=g, dtype=torch.int32)
    lens = torch.tensor([n, n // 2], dtype=torch.int32)
    q = torch.randint(-1, 2, (2, 4, 8), generator=g).to(BF16)
    for keep in (3, n // 3, n - 1, n + 4):
        got = ops.paged_kv_select(q.cuda(), bounds.cuda(), table.cuda(), lens.cuda(), keep, block_size=1)
        assert torch.equal(got.cpu(), plain_select(q, bounds, table, lens, keep, 1, 1, 1))


def test_select_scores_that_are_no_numbers_rank_lowest(need_gpu):
    bounds = torch.zeros(6, 1, 2, 8, dtype=BF16)
    bounds[1, 0, :, 0] = math.nan
    bounds[2, 0, :, 0] = -math.inf
    bounds[3, 0, 0, 0], bounds[3, 0, 1, 0] = -1.0, math.inf
    bounds[4, 0, :, 0] = -5.0
    bounds[5] = -0.0
    q = torch.zeros(1, 1, 8, dtype=BF16)
    q[..., 0] = 1.0
    table, lens = torch.arange(6, dtype=torch.int32)[None], torch.tensor([6], dtype=torch.int32)
    for keep, want in ((1, [3]), (2, [0, 3]), (3, [0, 3, 5]), (4, [0, 3, 4, 5]), (5, [0, 2, 3, 4, 5]), (6, [0, 1, 2, 3, 4, 5])):
        got = ops.paged_kv_select(q.cuda(), bounds.cuda(), table.cuda(), lens.cuda(), keep, block_size=1, sink=0, recent=0)
        assert got[0, 0].tolist() == want


# ---- eviction -----------------------------------------------------------------------------------


def plain_evict(mass, table, lens, budget, block, sink, recent):
    B, W = table.shape
    t, m = torch.full((B, W), -1, dtype=torch.int32), torch.zeros(B, W)
    ev, at = t.clone(), t.clone()
    new, count = torch.zeros(B, dtype=torch.int32), torch.zeros(B, dtype=torch.int32)
    for b in range(B):
        tokens = max(0, min(int(lens[b]), W * block))
        n = -(-tokens // block)
        can = [int(table[b, j]) >= 0 for j in range(n)]
        stay = best(mass[b, :n].tolist(), can, budget, sink, recent)
        gone = [j for j in range(n) if can[j] and j not in set(stay)]
        t[b, : len(stay)], m[b, : len(stay)] = table[b, stay], mass[b, stay]
        ev[b, : len(gone)], at[b, : len(gone)] = table[b, gone], torch.tensor(gone, dtype=torch.int32)
        new[b], count[b] = sum(min(block, tokens - j * block) for j in stay), len(gone)
    return t, new, m, ev, at, count


def check_evict(mass, table, lens, budget, block, sink, recent):
    before = [x.cuda() for x in (mass, table, lens)]
    got = ops.paged_kv_evict(*before[:3], budget, block_size=block, sink=sink, recent=recent)
    for a, b, name in zip(got, plain_evict(mass, table, lens, budget, block, sink, recent), got._fields):
        assert torch.equal(torch.nan_to_num(a.cpu(), nan=-77.0), torch.nan_to_num(b, nan=-77.0)), name
    for x, y in zip(before, (mass, table, lens)):
        assert torch.equal(torch.nan_to_num(x.cpu(), nan=-77.0), torch.nan_to_num(y, nan=-77.0))


@pytest.mark.parametrize("budget,sink,recent", [(1, 0, 1), (5, 1, 2), (40, 4, 7), (100000, 1, 1)])
@pytest.mark.parametrize("block", [1, 16, 30])
def test_evict(need_gpu, budget, sink, recent, block):
    g = torch.Generator().manual_seed(budget + block)
    lens = torch.tensor([0, 1, 5 * block, 5 * block + 1, 200 * block - 1, 90 * block, 2**31 - 1, -4], dtype=torch.int32)
    table = torch.randint(0, 10**6, (8, 200), generator=g, dtype=torch.int32)
    mass = torch.randint(0, 9, (8, 200), generator=g).float()
    table[4, 7], table[5, 0], mass[5, 3], mass[5, 4], mass[6, 50] = -1, -3, math.nan, -0.0, math.inf
    check_evict(mass, table, lens, budget, block, sink, recent)


@pytest.mark.parametrize("n", [512, 513, 4095, 8193, 40001])
def test_evict_long_requests(need_gpu, n):
    g = torch.Generator().manual_seed(n)
    table = torch.randperm(2 * n, generator=g).to(torch.int32).view(2, n)
    for mass in (torch.rand(2, n, generator=g), torch.ones(2, n)):
        check_evict(mass, table, torch.tensor([n * 16 - 3, n * 8], dtype=torch.int32), n // 2, 16, 1, 3)


# ---- together, and as programs run them -----------------------------------------------------------


def test_steps_with_a_bounded_cache_and_offload(need_gpu):
    """Decode with mass, evict, move the evicted blocks out, decode on, bring them back: attention over both
    parts, joined by their log-sums, is attention over the whole cache."""
    q, kv, table, lens = make(30, [400, 200, 37], 16, 8, 2, 64, BF16)
    kvg, tg, lg, qg = kv.cuda(), table.cuda(), lens.cuda(), q.cuda()
    mass = torch.zeros(table.shape, device="cuda")
    for _ in range(3):
        whole, whole_lse = ops.paged_kv_attention(qg, kvg, tg, lg, mass=mass, return_lse=True)
    assert torch.allclose(mass.sum(1).cpu(), torch.full((3,), 24.0), atol=1e-4)
    e = ops.paged_kv_evict(mass, tg, lg, 8, block_size=16)
    assert e.evicted_count.tolist() == [17, 5, 0] and e.context_lens.tolist() == [128, 8 * 16 - 8, 37]
    ids = [e.evicted_blocks[b, : int(e.evicted_count[b])].cpu().numpy() for b in range(3)]
    host = [ops.paged_kv_gather(kvg, i) for i in ids]
    kept, kept_lse = ops.paged_kv_attention(qg, kvg, e.block_table, e.context_lens, return_lse=True)
    check_attention(q, kv, e.block_table.cpu(), e.context_lens.cpu(), kept, kept_lse)
    other = torch.zeros_like(kvg)
    for i, h in zip(ids, host):
        if len(i):
            ops.paged_kv_scatter(other, i, h)
    back, back_lse = ops.paged_kv_attention(qg, other, e.evicted_blocks, e.evicted_count * 16, return_lse=True)
    top = torch.logaddexp(kept_lse, back_lse)
    joined = (kept_lse - top).exp()[..., None] * kept + (back_lse - top).exp()[..., None] * back
    assert torch.allclose(top, whole_lse, atol=1e-4)
    # two roundings to bf16 of the parts and one of the whole
    assert ((joined - whole).abs() <= 2.0 ** -8 * (kept.abs() + back.abs() + whole.abs()) + 1e-4).all()


def test_evicted_blocks_go_to_the_host_and_come_back(need_gpu):
    """Two layers, cut by the mass that both add up; the blocks that leave are saved in the pooled data plane,
    their pages overwritten, then restored into other pages: attention over all parts is as before."""
    from pcie_pool_b200.adapters import PagedKVOffloader
    from pcie_pool_b200.parallel.engine import PoolEngine
    from pcie_pool_b200.utils.host_memory import PinnedHostBuffer

    layers = [make(32 + i, [400, 37, 200], 16, 8, 2, 64, BF16, pages_extra=40) for i in range(2)]
    table, lens = layers[0][2].cuda(), layers[0][3].cuda()
    kvs = []
    for q, kv, t, _ in layers:  # one table for all layers
        g = torch.zeros_like(kv).cuda()
        g[:, table.long()] = kv.cuda()[:, t.cuda().long()].nan_to_num(0.0)
        kvs.append(g)
    qs = [x[0].cuda() for x in layers]
    mass = torch.zeros(table.shape, device="cuda")
    whole = [ops.paged_kv_attention(q, kv, table, lens, mass=mass, return_lse=True) for q, kv in zip(qs, kvs)]
    host = PinnedHostBuffer(1 << 20)
    try:
        store = PagedKVOffloader(PoolEngine([0], slot_bytes=1 << 20, slots=3, timeout_s=10.0), kvs, target=0)
        e, gone = store.evict(mass, table, lens, 6, host.ptr, 1 << 20, block_size=16)
        assert [(x.request, len(x.blocks)) for x in gone] == [(0, 19), (2, 7)]
        free = [p for x in gone for p in x.blocks][::-1]
        back = torch.full_like(table, -1)
        for kv in kvs:
            kv[:, free] = float("nan")  # the pages are used for something else
        for x in gone:
            pages, free = free[: len(x.blocks)], free[len(x.blocks):]
            store.restore(pages, host.ptr, 1 << 20, host_off=x.host_off)
            back[x.request, : len(pages)] = torch.tensor(pages, dtype=torch.int32)
    finally:
        host.release()
    torch.cuda.synchronize()
    for q, kv, (ref, ref_lse) in zip(qs, kvs, whole):
        kept, kept_lse = ops.paged_kv_attention(q, kv, e.block_table, e.context_lens, return_lse=True)
        rest, rest_lse = ops.paged_kv_attention(q, kv, back, e.evicted_count * 16, return_lse=True)
        top = torch.logaddexp(kept_lse, rest_lse)
        joined = (kept_lse - top).exp()[..., None] * kept + (rest_lse - top).exp()[..., None] * rest
        assert torch.allclose(top, ref_lse, atol=1e-4)
        # two roundings to bf16 of the parts and one of the whole
        assert ((joined - ref).abs() <= 2.0 ** -8 * (kept.abs() + rest.abs() + ref.abs()) + 1e-4).all()


def test_steps_with_sparse_reads(need_gpu):
    """A cache that grows by a token a step, its bounds kept up, blocks selected and read, against the plain forms."""
    q, kv, table, lens = make(31, [300, 158, 31], 16, 8, 2, 64, BF16)
    for b in range(3):  # the places of the next steps
        n = int(lens[b])
        for t in range(n, n + 4):
            kv[:, table[b, t // 16], t % 16] = torch.randn(2, 2, 64).to(BF16)
    table[1, 10] = kv.shape[1] - 1
    kv[:, -1] = torch.randn(2, 16, 2, 64).to(BF16)
    kvg, tg, qg = kv.cuda(), table.cuda(), q.cuda()
    bounds = torch.zeros(kv.shape[1], 2, 2, 64, dtype=BF16, device="cuda")
    ops.paged_kv_bounds(kvg, tg, lens.cuda(), bounds)
    for step in range(1, 4):
        now = lens + step
        ops.paged_kv_bounds(kvg, tg, now.cuda(), bounds, new_tokens=1)
        blocks = ops.paged_kv_select(qg, bounds, tg, now.cuda(), 6, block_size=16, sink=1, recent=2)
        ref = plain_bounds(kv, table, now, torch.zeros_like(bounds.cpu()), None)
        assert torch.equal(blocks.cpu(), plain_select(q, ref, table, now, 6, 16, 1, 2))
        out, lse = ops.paged_kv_attention(qg, kvg, tg, now.cuda(), blocks=blocks, return_lse=True)
        check_attention(q, kv, table, now, out, lse, blocks=blocks.cpu())


def one_step(s):
    out, lse = ops.paged_kv_attention(s["q"], s["kv"], s["table"], s["lens"], mass=s["mass"], return_lse=True)
    ops.paged_kv_bounds(s["kv"], s["table"], s["lens"], s["bounds"])
    blocks = ops.paged_kv_select(s["q"], s["bounds"], s["table"], s["lens"], 5, block_size=16)
    some = ops.paged_kv_attention(s["q"], s["kv"], s["table"], s["lens"], blocks=blocks)
    e = ops.paged_kv_evict(s["mass"], s["table"], s["lens"], 4, block_size=16)
    return [out, lse, s["mass"], s["bounds"], blocks, some, *e]


def fresh(seed, lens=(300, 0, 77, 1500)):
    q, kv, table, lens = (t.cuda() for t in make(seed, list(lens), 16, 8, 2, 64, BF16))
    return dict(q=q, kv=kv, table=table, lens=lens, mass=torch.zeros(table.shape, device="cuda"),
                bounds=torch.zeros(kv.shape[1], 2, 2, 64, dtype=BF16, device="cuda"))


def same(a, b):
    return all(torch.equal(torch.nan_to_num(x.float(), nan=3e38), torch.nan_to_num(y.float(), nan=3e38)) for x, y in zip(a, b))


def test_captured_replayed_with_other_contents(need_gpu):
    a, b = fresh(40), fresh(41)
    one_step(fresh(40))
    torch.cuda.synchronize()
    graphs, outs = [], []
    for s in (a, b):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(one_step(s))
        graphs.append(g)
    # two graphs of two states at once, on two streams
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(5):
        for s in (a, b):
            s["mass"].zero_()
        torch.cuda.synchronize()
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize()
        assert same(outs[0], one_step(fresh(40))) and same(outs[1], one_step(fresh(41)))
    # other lengths and values in the same places
    c = fresh(42, (17, 1490, 290, 0))
    for k in ("q", "lens"):
        a[k].copy_(c[k])
    a["table"].fill_(-1)
    w = min(a["table"].shape[1], c["table"].shape[1])
    a["table"][:, :w], a["kv"][:, : c["kv"].shape[1]] = c["table"][:, :w], c["kv"][:, : a["kv"].shape[1]]
    a["mass"].zero_()
    a["bounds"].zero_()
    d = {k: v.clone() for k, v in a.items()}
    graphs[0].replay()
    torch.cuda.synchronize()
    assert same(outs[0], one_step(d))


def test_first_call_of_a_process_may_be_captured(need_gpu):
    import subprocess
    import sys
    from pathlib import Path

    code = """
import torch
from tests.test_gpu_paged_kv import fresh, one_step, same
s = fresh(40)
g = torch.cuda.CUDAGraph()
torch.cuda.synchronize()
with torch.cuda.graph(g):
    out = one_step(s)
g.replay()
torch.cuda.synchronize()
assert same(out, one_step(fresh(40)))
print("captured")
"""
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300,
                       cwd=Path(__file__).resolve().parents[1])
    assert r.returncode == 0 and "captured" in r.stdout, r.stderr[-3000:]


def test_calls_on_two_streams_at_once(need_gpu):
    states = [fresh(50 + i) for i in range(4)]
    want = [one_step(fresh(50 + i)) for i in range(4)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(4)]
    for _ in range(10):
        for s in states:
            s["mass"].zero_()
        torch.cuda.synchronize()
        got = []
        for s, st in zip(states, streams):
            with torch.cuda.stream(st):
                got.append(one_step(s))
        torch.cuda.synchronize()
        assert all(same(x, y) for x, y in zip(got, want))


def test_another_device_than_the_current(need_two_gpus):
    want = one_step(fresh(60))
    s = {k: v.to("cuda:1") for k, v in fresh(60).items()}
    assert torch.cuda.current_device() == 0
    got = one_step(s)
    torch.cuda.synchronize(1)
    assert same([x.cpu() for x in got], [x.cpu() for x in want]) and torch.cuda.current_device() == 0


def test_tensors_on_two_devices_are_refused(need_gpu):
    s = fresh(61)
    with pytest.raises(ValueError, match="one CUDA device"):
        ops.paged_kv_attention(s["q"], s["kv"], s["table"].cpu(), s["lens"])
    with pytest.raises(ValueError, match="device"):
        ops.paged_kv_attention(s["q"].cpu(), s["kv"], s["table"], s["lens"])
