"""Inputs and 64-bit oracles shared by the paged-KV tests."""

import math

import torch


def make(seed, lens, block, heads, kv_heads, dim, dtype, pages_extra=3, layout="planes", width_extra=1):
    """CPU tensors (q, kv, table, lens): a cache whose unused places hold NaN, and a table whose entries
    behind a request's last block point anywhere."""
    g = torch.Generator().manual_seed(seed)
    need = [-(-max(n, 0) // block) for n in lens]
    pages, width = sum(need) + pages_extra, max(need, default=0) + width_extra
    kv = torch.full((2, pages, block, kv_heads, dim), math.nan, dtype=dtype)
    table = torch.randint(0, pages, (len(lens), width), generator=g, dtype=torch.int32)
    order = torch.randperm(pages, generator=g).to(torch.int32)
    at = 0
    for b, n in enumerate(lens):
        table[b, : need[b]] = order[at: at + need[b]]
        for j in range(need[b]):
            m = min(block, n - j * block)
            kv[:, table[b, j], :m] = torch.randn(2, m, kv_heads, dim, generator=g).to(dtype)
        at += need[b]
    q = (torch.randn(len(lens), heads, dim, generator=g) * 1.5).to(dtype)
    if layout == "pages":     # [pages, 2, block, heads, dim]
        kv = kv.transpose(0, 1).contiguous().transpose(0, 1)
    elif layout == "heads":   # [2, pages, heads, block, dim]
        kv = kv.transpose(2, 3).contiguous().transpose(2, 3)
    elif layout == "padded":  # rows of a wider buffer
        wide = torch.full((2, pages, block, kv_heads, dim + 16), math.nan, dtype=dtype)
        wide[..., 8: 8 + dim] = kv
        kv = wide[..., 8: 8 + dim]
    return q, kv, table, torch.tensor(lens, dtype=torch.int32)


def to_gpu(kv):
    """On the GPU with the same strides."""
    out = torch.empty_strided(kv.size(), kv.stride(), dtype=kv.dtype, device="cuda")
    return out.copy_(kv)


def attention(q, kv, table, lens, scale=None, blocks=None):
    """(out, lse, weight of each block, bound on the error of out) in 64 bits."""
    B, H, D = q.shape
    pages, bs, Hk = kv.shape[1:4]
    scale = D ** -0.5 if scale is None else scale
    out, err = torch.zeros(B, H, D, dtype=torch.float64), torch.zeros(B, H, D, dtype=torch.float64)
    lse = torch.full((B, H), -math.inf, dtype=torch.float64)
    lse_err = torch.zeros(B, H, dtype=torch.float64)
    weight = torch.zeros(table.shape, dtype=torch.float64)
    u = 2.0 ** -24
    for b in range(B):
        n = max(0, min(int(lens[b]), table.shape[1] * bs))
        m = -(-n // bs)
        for h in range(H):
            g = h // (H // Hk)
            js = range(m) if blocks is None else [int(j) for j in blocks[b, g, :m]]
            k, v, owner = [], [], []
            for j in js:
                if not 0 <= j < m or not 0 <= int(table[b, j]) < pages:
                    continue
                t = min(bs, n - j * bs)
                k.append(kv[0, table[b, j], :t, g].double())
                v.append(kv[1, table[b, j], :t, g].double())
                owner += [j] * t
            if not k:
                continue
            k, v, x = torch.cat(k), torch.cat(v), q[b, h].double()
            s = (k @ x) * scale
            lse[b, h] = s.logsumexp(0)
            p = (s - lse[b, h]).exp()
            out[b, h] = p @ v
            weight[b].index_add_(0, torch.tensor(owner), p)
            # a score is a sum of dim products, scaled: dim + 3 roundings, two more where it is taken to base 2 and
            # its maximum is subtracted; a weight is off by that twice (its own and the sum's), by exp2's 2^-22, and by
            # 2^-16 where it is split into two numbers of 8 bits; sums over n weights round n times at most
            ds = float(((k.abs() @ x.abs()).max() * abs(scale) * (D + 3) + 4 * s.abs().max()) * u)
            lse_err[b, h] = ds + len(owner) * u + 2.0 ** -21 + 2 * u * abs(lse[b, h])
            err[b, h] = (2 * ds + (2 * len(owner) + 64) * u + 2.0 ** -16 + 2.0 ** -20) * (p @ v.abs())
    return out, lse, weight, err, lse_err


def best(values, can, keep, sink, recent):
    """Indices, ascending, of the ``keep`` highest among ``can``: first and last ones first, NaN lowest."""
    n = len(values)

    def rank(j):
        if j < sink or j >= n - recent:
            return (0, 0.0, j)
        v = values[j]
        return (2, 0.0, j) if v != v else (1, -v, j)

    return sorted(sorted((j for j in range(n) if can[j]), key=rank)[:keep])


def scores(q, bounds, rows):
    """fp32 scores [Hk, len(rows)] of rows of ``bounds``: the group's sum of upper bounds, rounded once."""
    H, D = q.shape
    Hk = bounds.shape[1]
    out = torch.zeros(Hk, len(rows), dtype=torch.float64)
    for g in range(Hk):
        lo, hi = bounds[rows, g].double().unbind(1)
        for x in q[g * H // Hk: (g + 1) * H // Hk].double():
            out[g] += torch.maximum(x * lo, x * hi).sum(1)
    return out.float()
