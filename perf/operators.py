"""Cases of the paged-KV operators: attention of one new token over a paged cache
(with the attention mass of its blocks), sparse attention over blocks that their
key bounds select, the bounds themselves, and eviction by accumulated mass.

``run`` computes a case in plain torch operations, or with ``own`` set through
``pcie_pool_b200.ops``.  The cache of one layer is ``[2, pages, block, kv_heads,
dim]`` (K, then V); ``pages`` of it are in use, in random order.
"""

import math

import torch

own = False

LLAMA = dict(heads=32, kv_heads=8, dim=128, block=16, dtype="bf16")   # the 8B decoder's cache layer
DECODER_7B = dict(heads=32, kv_heads=32, dim=128, block=16, dtype="fp16")  # one key head for each query head


def listed():
    return [
        # one chat request, short context: the latency of a call
        dict(LLAMA, name="attend_one_request", op="attend", requests=1, tokens=300, ragged=False, idle=0,
             mass=False, pages_first=False),
        # a serving batch: lengths from tens to thousands, two slots of the batch empty
        dict(LLAMA, name="attend_batch", op="attend", requests=64, tokens=8192, ragged=True, idle=2,
             mass=False, pages_first=False),
        # the offload benchmark's eight requests of 32k tokens
        dict(LLAMA, name="attend_32k", op="attend", requests=8, tokens=32768, ragged=False, idle=0,
             mass=False, pages_first=False),
        # as many key heads as query heads, fp16, K and V of a page next to each other
        dict(DECODER_7B, name="attend_7b_fp16", op="attend", requests=16, tokens=4000, ragged=True, idle=0,
             mass=False, pages_first=True),
        # a batch that also gathers the attention mass of its blocks, to choose what to offload
        dict(LLAMA, name="attend_mass_batch", op="attend", requests=32, tokens=8192, ragged=True, idle=1,
             mass=True, pages_first=False),
        # a small decoder: few heads, odd length, larger pages
        dict(heads=10, kv_heads=2, dim=64, block=32, dtype="fp16", name="attend_mass_small", op="attend",
             requests=3, tokens=1237, ragged=True, idle=0, mass=True, pages_first=False),
        # one very long request: an eighth of its blocks is chosen and read
        dict(LLAMA, name="sparse_128k", op="sparse", requests=1, tokens=131072, ragged=False, idle=0, keep=1024,
             sink=1, recent=4),
        # long requests in a batch, each reads at most 128 blocks
        dict(LLAMA, name="sparse_batch", op="sparse", requests=16, tokens=32768, ragged=True, idle=1, keep=128,
             sink=1, recent=2),
        # bounds of whole prompts after they were restored or computed
        dict(LLAMA, name="bounds_prompts", op="bounds", requests=8, tokens=32768, ragged=True, idle=0, new_tokens=0),
        # bounds of the blocks that the last token went to, every step of a batch
        dict(LLAMA, name="bounds_step", op="bounds", requests=64, tokens=8192, ragged=True, idle=2, new_tokens=1),
        # a batch of long requests is cut to half of its longest
        dict(name="evict_batch", op="evict", requests=64, tokens=32768, block=16, ragged=True, idle=2, budget=1024,
             sink=1, recent=4),
        # one short request
        dict(name="evict_one", op="evict", requests=1, tokens=1500, block=16, ragged=False, idle=0, budget=32,
             sink=1, recent=2),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attend", "attend", "sparse", "bounds", "evict"])
    c = dict(op=op, requests=_log(rng, 1, 96), tokens=_log(rng, 1, 131072), ragged=rng.random() < 0.7,
             block=rng.choice([16, 16, 32, 64]))
    c["idle"] = rng.choice([0, 0, 1, 2]) if c["requests"] > 4 else 0
    if op == "evict":
        c["tokens"] = min(c["tokens"], 2_000_000 // c["requests"])
        c["sink"], c["recent"] = rng.choice([0, 1, 4]), rng.choice([1, 2, 7])
        blocks = -(-c["tokens"] // c["block"])
        c["budget"] = max(c["sink"] + c["recent"], int(blocks * rng.uniform(0.1, 0.9)))
        return c
    heads, kv_heads = rng.choice([(32, 8), (32, 8), (32, 32), (10, 2), (8, 1), (40, 8), (28, 4), (24, 1), (16, 1)])
    c.update(heads=heads, kv_heads=kv_heads, dim=rng.choice([128, 128, 128, 64, 96, 256]), dtype=rng.choice(["bf16", "fp16"]))
    if op != "sparse" and not c["ragged"]:
        c["block"] = rng.choice([16, 8, 24, 128])
    c["tokens"] = max(1, min(c["tokens"], 250_000_000 // (c["requests"] * kv_heads * c["dim"])))
    blocks = -(-c["tokens"] // c["block"])
    if op == "attend":
        c["mass"] = rng.random() < 0.4 and c["block"] % 16 == 0
        c["pages_first"] = rng.random() < 0.3
    elif op == "sparse":
        c["sink"], c["recent"] = rng.choice([0, 1, 4]), rng.choice([1, 2, 7])
        c["keep"] = max(c["sink"] + c["recent"], min(blocks, _log(rng, 1, 1024)))
    else:
        c["new_tokens"] = rng.choice([0, 0, 1, 1, 5, 200])
    return c


def _lens(case):
    """The requests' lengths, from the case alone: log-spaced below ``tokens`` and out of order where
    ragged, with the last ``idle`` slots empty."""
    n, most = case["requests"], case["tokens"]
    lens = [most] * n
    if case["ragged"] and n > 1:
        low = max(1.0, most ** 0.5)
        at = sorted(range(n), key=lambda i: (i * 0.6180339887) % 1.0)
        lens = [int(round(low * (most / low) ** (k / (n - 1)))) for k in at]
    return [0 if i >= n - case["idle"] else v for i, v in enumerate(lens)]


def _dtype(case):
    return {"bf16": torch.bfloat16, "fp16": torch.float16}[case["dtype"]]


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    lens, bs = _lens(case), case["block"]
    need = [-(-v // bs) for v in lens]
    width, pages = max(need), sum(need) + 5
    s = dict(case=case, lens=torch.tensor(lens, dtype=torch.int32, device=dev))
    # pages of a request are wherever they were free; entries behind a request's last page are left from others
    order = torch.randperm(pages, device=dev, generator=g).to(torch.int32)
    table = torch.randint(0, pages, (len(lens), width), device=dev, generator=g, dtype=torch.int32)
    at = torch.arange(width, device=dev)[None, :] < torch.tensor(need, device=dev)[:, None]
    table[at] = order[: sum(need)]
    s["table"] = table
    if case["op"] == "evict":
        # accumulated weight is heavy-tailed: a few blocks hold most of it; some never got any
        m = torch.randn(table.shape, device=dev, generator=g).mul_(2).exp_()
        m *= torch.rand(table.shape, device=dev, generator=g) > 0.05
        s["mass"] = m
        return s
    dt, hk, d = _dtype(case), case["kv_heads"], case["dim"]
    shape = (pages, 2, bs, hk, d) if case.get("pages_first") else (2, pages, bs, hk, d)
    kv = torch.randn(shape, device=dev, generator=g, dtype=dt)
    s["kv"] = kv.transpose(0, 1) if case.get("pages_first") else kv
    # keys have channels that carry more than others
    s["kv"][0] *= (1 + torch.rand(hk, d, device=dev, generator=g)).to(dt)
    s["q"] = (torch.randn(len(lens), case["heads"], d, device=dev, generator=g) * 1.5).to(dt)
    if case.get("mass"):
        s["mass"] = torch.rand(table.shape, device=dev, generator=g)
    if case["op"] == "sparse":
        s["bounds"] = torch.stack((s["kv"][0].amin(1), s["kv"][0].amax(1)), 2).contiguous()
        # the last page of a request is not full: its bounds are those of the filled part
        s["bounds"] = _bounds(s["kv"][0], table, s["lens"], s["bounds"], 0)
    if case["op"] == "bounds":
        s["bounds"] = torch.zeros(pages, hk, 2, d, device=dev, dtype=dt)
    return s


# ---- plain forms -----------------------------------------------------------------------


def _attend(q, k, v, pages, pos, lens, mass):
    """q [B, Hk, G, D]; k, v [pages, block, Hk, D]; pages, pos [B, Hk or 1, n]: the page of a slot and its first position."""
    b, hk, _, d = q.shape
    bs = k.shape[1]
    pos = pos[..., None] + torch.arange(bs, device=q.device)
    ok = ((pos < lens[:, None, None, None]) & (pages >= 0)[..., None]).flatten(2)[:, :, None]
    at = pages.clamp(min=0).long()
    if pages.shape[1] == 1:  # one list for all key heads
        k, v = (x[at[:, 0]].flatten(1, 2).transpose(1, 2).float() for x in (k, v))
    else:
        heads = torch.arange(hk, device=q.device)[None, :, None]
        k, v = (x.transpose(1, 2)[at, heads].flatten(2, 3).float() for x in (k, v))
    s = (q.float() @ k.transpose(2, 3)) / math.sqrt(d)
    s = torch.where(ok, s, -math.inf)
    top = s.amax(3, keepdim=True).clamp(min=-1e30)
    e = (s - top).exp()
    total = e.sum(3, keepdim=True)
    p = e / total.clamp(min=1e-30)
    out = p @ torch.where(ok.transpose(2, 3), v, 0.0)
    if mass is not None:
        mass += p.sum((1, 2)).unflatten(1, (-1, bs)).sum(2)
    return out, (top + total.log())[..., 0]


def _bounds(k, table, lens, bounds, new_tokens):
    bs = k.shape[1]
    first = torch.arange(table.shape[1], device=k.device)[None, :] * bs
    since = (lens - new_tokens).clamp(min=0) if new_tokens else lens * 0
    todo = (first < lens[:, None]) & (first + bs > since[:, None])
    rows = table[todo].long()
    ok = ((first[..., None] + torch.arange(bs, device=k.device)) < lens[:, None, None])[todo][:, :, None, None]
    keys = k[rows].float()
    lo = torch.where(ok, keys, math.inf).amin(1)
    hi = torch.where(ok, keys, -math.inf).amax(1)
    bounds[rows] = torch.stack((lo, hi), 2).to(k.dtype)
    return bounds


def _keep(score, can, must, keep):
    """The ``keep`` highest of the last axis among ``can``, those of ``must`` first, ties to the lowest index, ascending; -1 behind."""
    n, can = score.shape[-1], can.expand_as(score)
    rank = torch.where(can, torch.where(must, math.inf, score), -math.inf)
    # two stable sorts: by score, then what cannot be taken behind what can
    order = torch.sort(rank, dim=-1, descending=True, stable=True).indices
    later = torch.sort((~can).gather(-1, order).to(torch.int32), dim=-1, stable=True).indices
    order = order.gather(-1, later)[..., :keep]
    taken = can.gather(-1, order)
    found = torch.where(taken, order, n).sort(-1).values
    found = torch.where(found < n, found, -1).to(torch.int32)
    return torch.nn.functional.pad(found, (0, max(0, keep - n)), value=-1)


def _select(q, bounds, table, lens, case):
    """q [B, Hk, G, D].  The score's sums are taken in 64 bits and rounded once, so that the order does not hang on their order."""
    b = bounds[table.clamp(min=0).long()].double()
    score = (q.double().clamp(min=0).sum(2)[:, None] * b[..., 1, :]).sum(3)
    score = score + (q.double().clamp(max=0).sum(2)[:, None] * b[..., 0, :]).sum(3)
    return _keep(score.transpose(1, 2).float(), *_can_must(table, lens, case, 1), case["keep"])


def _can_must(table, lens, case, heads):
    j = torch.arange(table.shape[1], device=table.device)[None]
    n = ((lens + case["block"] - 1) // case["block"])[:, None]
    can = (j < n) & (table >= 0)
    must = (j < case["sink"]) | (j >= n - case["recent"])
    return (can[:, None], must[:, None]) if heads else (can, must)


def _evict(mass, table, lens, case):
    bs, width = case["block"], table.shape[1]
    can, must = _can_must(table, lens, case, 0)
    kept = _keep(mass, can, must, case["budget"])[:, :width]
    kept = torch.nn.functional.pad(kept, (0, width - kept.shape[1]), value=-1)
    at = kept.clamp(min=0).long()
    stays = torch.zeros_like(can).scatter_(1, at, kept >= 0) if width else can
    # scatter_ of the padding's entries may clear index 0: set it from the list itself
    stays[:, 0] = kept[:, 0] == 0
    pos = torch.arange(width, device=table.device)[None]
    gone = torch.where(can & ~stays, pos, width).sort(1).values
    gone = torch.where(gone < width, gone, -1).to(torch.int32)
    last = (lens[:, None] - kept * bs).clamp(max=bs)
    return dict(
        table=torch.where(kept >= 0, table.gather(1, at), -1),
        lens=torch.where(kept >= 0, last, 0).sum(1).to(torch.int32),
        mass=torch.where(kept >= 0, mass.gather(1, at), 0.0),
        pages=torch.where(gone >= 0, table.gather(1, gone.clamp(min=0).long()), -1),
        index=gone,
        count=(gone >= 0).sum(1).to(torch.int32),
    )


def _run_plain(s):
    case, table, lens = s["case"], s["table"], s["lens"]
    if case["op"] == "evict":
        return _evict(s["mass"], table, lens, case)
    k, v = s["kv"][0], s["kv"][1]
    if case["op"] == "bounds":
        return _bounds(k, table, lens, s["bounds"], case["new_tokens"])
    b, h, d = s["q"].shape
    q = s["q"].view(b, case["kv_heads"], -1, d)
    if case["op"] == "attend":
        first = torch.arange(table.shape[1], device=table.device)[None, None] * case["block"]
        out, lse = _attend(q, k, v, table[:, None], first, lens, s.get("mass"))
        r = dict(out=out.reshape(b, h, d).to(s["q"].dtype), lse=lse.reshape(b, h))
        return dict(r, mass=s["mass"]) if case["mass"] else r
    blocks = _select(q, s["bounds"], table, lens, case)
    at = blocks.clamp(min=0).long()
    pages = torch.where(blocks >= 0, table[:, None].expand(-1, blocks.shape[1], -1).gather(2, at), -1)
    out, lse = _attend(q, k, v, pages, at * case["block"], lens, None)
    return dict(out=out.reshape(b, h, d).to(s["q"].dtype), lse=lse.reshape(b, h), blocks=blocks)


def _run_own(s):
    from pcie_pool_b200 import ops

    case, table, lens = s["case"], s["table"], s["lens"]
    if case["op"] == "evict":
        e = ops.paged_kv_evict(s["mass"], table, lens, case["budget"], block_size=case["block"], sink=case["sink"],
                               recent=case["recent"])
        return dict(table=e.block_table, lens=e.context_lens, mass=e.mass, pages=e.evicted_blocks,
                    index=e.evicted_index, count=e.evicted_count)
    if case["op"] == "bounds":
        return ops.paged_kv_bounds(s["kv"], table, lens, s["bounds"], new_tokens=case["new_tokens"] or None)
    if case["op"] == "attend":
        out, lse = ops.paged_kv_attention(s["q"], s["kv"], table, lens, mass=s.get("mass"), return_lse=True)
        r = dict(out=out, lse=lse)
        return dict(r, mass=s["mass"]) if case["mass"] else r
    blocks = ops.paged_kv_select(s["q"], s["bounds"], table, lens, case["keep"], block_size=case["block"],
                                 sink=case["sink"], recent=case["recent"])
    out, lse = ops.paged_kv_attention(s["q"], s["kv"], table, lens, blocks=blocks, return_lse=True)
    return dict(out=out, lse=lse, blocks=blocks)


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---- work --------------------------------------------------------------------------------


def work(case):
    lens, bs = _lens(case), case["block"]
    blocks = [-(-v // bs) for v in lens]
    if case["op"] == "evict":
        # reads mass and table of the blocks in use; writes both tables, the lists of what left, lengths and counts
        width = max(blocks)
        return {"bytes": 8 * sum(blocks) + 16 * width * len(lens) + 12 * len(lens), "flops": 0}
    token = case["kv_heads"] * case["dim"] * 2  # bytes of a token's keys
    if case["op"] == "bounds":
        new = case["new_tokens"]
        done = [0 if not new else max(0, v - new) // bs for v in lens]
        read = sum(v - f * bs for v, f in zip(lens, done))
        wrote = sum(b - f for b, f in zip(blocks, done) if b > f)
        return {"bytes": read * token + wrote * 2 * token + 4 * (wrote + len(lens)), "flops": 2 * read * token // 2}
    used, extra, flops = lens, 0, 0
    if case["op"] == "sparse":
        used = [min(v, case["keep"] * bs) for v in lens]
        extra = sum(blocks) * 2 * token + 4 * len(lens) * case["kv_heads"] * case["keep"]
        flops = sum(blocks) * 2 * token
    elif case["mass"]:
        extra = 8 * sum(blocks)
    rows = len(lens) * case["heads"]
    return {"bytes": sum(used) * 2 * token + rows * (case["dim"] * 4 + 4) + 4 * (sum(blocks) + len(lens)) + extra,
            "flops": flops + 4 * case["heads"] * case["dim"] * sum(used)}


# ---- in 64 bits ----------------------------------------------------------------------------


def _best(values, keep, sink, recent):
    """Indices, ascending, of the ``keep`` highest of a list in Python, ties to the lowest."""
    n = len(values)
    must = [j for j in range(n) if j < sink or j >= n - recent]
    rest = sorted((j for j in range(n) if not (j < sink or j >= n - recent)), key=lambda j: (-values[j], j))
    return sorted((must + rest)[:keep])


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] in ("evict", "bounds"):
        return _exact_lists(case, s)
    lens, bs, hk, d = _lens(case), case["block"], case["kv_heads"], case["dim"]
    b, h = len(lens), case["heads"]
    out = torch.zeros(b, h, d, dtype=torch.float64, device="cuda")
    lse = torch.full((b, h), -math.inf, dtype=torch.float64, device="cuda")
    mass = s["mass"].double() if case.get("mass") else None
    chosen = torch.full((b, hk, case.get("keep", 0)), -1, dtype=torch.int32)
    for i, n in enumerate(lens):
        if not n:
            continue
        m = -(-n // bs)
        pages = s["table"][i, :m].long()
        for j in range(hk):
            q = s["q"][i, j * h // hk:(j + 1) * h // hk].double()
            mine = torch.arange(m, device="cuda")
            if case["op"] == "sparse":
                lo, hi = s["bounds"][pages, j].double().unbind(1)
                bound = sum(torch.maximum(x * lo, x * hi).sum(1) for x in q).float().tolist()
                at = _best(bound, case["keep"], case["sink"], case["recent"])
                chosen[i, j, :len(at)] = torch.tensor(at)
                mine = torch.tensor(at, device="cuda")
            where = (mine[:, None] * bs + torch.arange(bs, device="cuda")).flatten()
            keys, values = (x[pages[mine], :, j].flatten(0, 1)[where < n].double() for x in s["kv"])
            logits = keys @ q.T * d ** -0.5
            lse[i, j * h // hk:(j + 1) * h // hk] = logits.logsumexp(0)
            w = logits.softmax(0)
            out[i, j * h // hk:(j + 1) * h // hk] = w.T @ values
            if mass is not None:
                mass[i].index_add_(0, where[where < n] // bs, w.sum(1))
    r = dict(out=out, lse=lse)
    if mass is not None:
        r["mass"] = mass
    return dict(r, blocks=chosen) if case["op"] == "sparse" else r


def _exact_lists(case, s):
    lens, bs = _lens(case), case["block"]
    table = s["table"].tolist()
    if case["op"] == "bounds":
        b = s["bounds"].double()
        for i, n in enumerate(lens):
            start = max(0, n - case["new_tokens"]) // bs if case["new_tokens"] else 0
            full = n // bs
            if full > start:
                k = s["kv"][0][s["table"][i, start:full].long()].double()
                b[s["table"][i, start:full].long()] = torch.stack((k.min(1).values, k.max(1).values), 2)
            if n > full * bs:
                k = s["kv"][0][table[i][full], : n - full * bs].double()
                b[table[i][full]] = torch.stack((k.min(0).values, k.max(0).values), 1)
        return b
    width = len(table[0])
    mass = s["mass"].tolist()
    new = {k: [] for k in ("table", "lens", "mass", "pages", "index", "count")}
    fill = lambda v, x: v + [x] * (width - len(v))  # noqa: E731
    for i, n in enumerate(lens):
        m = -(-n // bs)
        stay = _best(mass[i][:m], case["budget"], case["sink"], case["recent"]) if m > case["budget"] else list(range(m))
        gone = sorted(set(range(m)) - set(stay))
        new["table"].append(fill([table[i][j] for j in stay], -1))
        new["mass"].append(fill([mass[i][j] for j in stay], 0.0))
        new["lens"].append(sum(min(bs, n - j * bs) for j in stay))
        new["pages"].append(fill([table[i][j] for j in gone], -1))
        new["index"].append(fill(gone, -1))
        new["count"].append(len(gone))
    return {k: torch.tensor(v, dtype=torch.float64 if k == "mass" else torch.int32) for k, v in new.items()}
