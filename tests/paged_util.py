"""Plain 64-bit forms of the serving operators, and caches to try them on."""
import math

import torch


def make_cache(b, hk, d, lengths, page, sets=1, dtype=torch.bfloat16, seed=0, std=1., garbage=float('nan'), spare=3, width=None):
    """Pools in which the sequences' pages lie in no order.  Every row that belongs to no sequence holds ``garbage``."""
    g = torch.Generator().manual_seed(seed)
    width = max(1, max(-(-n // page) for n in lengths)) if width is None else width
    pages = b * width + spare
    tables = torch.randperm(pages, generator=g)[:b * width].view(b, width).to(torch.int32)
    pools = []
    for _ in range(2 * sets):
        pool = torch.full((pages, page, hk, d), garbage)
        for s, n in enumerate(lengths):
            n = max(0, min(n, width * page))
            x = torch.arange(n)
            pool[tables[s].long()[x // page], x % page] = torch.randn(n, hk, d, generator=g) * std
        pools.append(pool.to(dtype).cuda())
    return pools, tables.cuda()


def rows_of(pool, table, count):
    """Rows of positions 0 .. count - 1 in 64 bits, and which of them are there."""
    page = pool.shape[1]
    x = torch.arange(count, device=pool.device)
    there = x < len(table) * page
    entry = table.long()[(x // page).clamp(max=max(len(table) - 1, 0))] if len(table) else torch.full_like(x, -1)
    there = there & (entry >= 0) & (entry < pool.shape[0])
    return pool[entry.clamp(0, pool.shape[0] - 1), x % page].double(), there


def attend(q, keys, values, tables, lengths, counts=None, w1=None, w2=None, scale=None):
    """Dense (one set) or 2-simplicial (two sets) attention of every row, row by row, from the definition."""
    b, n, h, d = q.shape
    hk = keys[0].shape[2]
    scale = d ** -0.5 if scale is None else scale
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    for s in range(b):
        length = max(int(lengths[s]), 0)
        count = n if counts is None else min(max(int(counts[s]), 0), n)
        if length == 0:
            continue
        kv = [rows_of(p, tables[s], length) for p in (*keys, *values)]
        there = kv[0][1]
        kv = [r[..., :d] for r, _ in kv]
        for t in range(count):
            p = length - count + t
            if p < 0:
                continue
            for hh in range(h):
                z = hh // (h // hk)
                qq = q[s, t, hh].double() * scale
                if len(keys) == 1:
                    j = torch.nonzero(there[:p + 1])[:, 0]
                    if len(j):
                        a = torch.softmax(kv[0][j, z] @ qq, 0)
                        out[s, t, hh] = a @ kv[1][j, z]
                    continue
                lo1, lo2 = max(0, p - w1 + 1), max(0, p - w2 + 1)
                j = torch.nonzero(there[lo1:p + 1])[:, 0] + lo1
                k = torch.nonzero(there[lo2:p + 1])[:, 0] + lo2
                if len(j) and len(k):
                    x = (kv[1][k, z] * qq) @ kv[0][j, z].T
                    a = torch.softmax(x.flatten(), 0).view_as(x)
                    out[s, t, hh] = ((a @ kv[2][j, z]) * kv[3][k, z]).sum(0)
    return out


# Roundings to the element type: the output, the weights of the second product and, in the 2-simplicial form, q * k2.  Each has a relative error of at most half an
# ulp (2^-9 in bf16, 2^-12 in fp16; rms 0.6 of that) and they are independent, so the norm of the error is below 3 * 2^-9 (2^-12) of the result's.  Elementwise the
# criterion of the other kernels of this package, and an eighth of it in fp16.
NORM = {torch.bfloat16: 3 * 2. ** -9, torch.float16: 3 * 2. ** -12}
ELEMENT = {torch.bfloat16: (2e-2, 1e-2), torch.float16: (2.5e-3, 1.25e-3)}


def check(got, want, dtype=None):
    dtype = got.dtype if dtype is None else dtype
    got = got.double()
    assert got.shape == want.shape
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    fine = ~torch.isnan(want)
    err = (got - want)[fine].abs()
    atol, rtol = ELEMENT[dtype]
    assert bool((err <= atol + rtol * want[fine].abs()).all()), float(err.max())
    norm = float(want[fine].norm())
    assert float(err.norm()) <= NORM[dtype] * norm + 1e-12, float(err.norm()) / max(norm, 1e-30)


def sample(logits, noise, temperature, top_k, top_p, min_p):
    """(token, logprob) of every row, from the definition."""
    tokens, logprobs = [], []
    for r in range(len(logits)):
        x = logits[r].double()
        x = torch.where(torch.isnan(x), -math.inf, x).clamp(max=torch.finfo(torch.float32).max)
        if bool((x == -math.inf).all()):
            tokens.append(-1)
            logprobs.append(-math.inf)
            continue
        order = torch.sort(x, descending=True, stable=True).indices
        token = int(order[0])
        if temperature[r] > 0:
            p = torch.softmax((x - x.max()) / temperature[r], -1)[order]
            keep = p >= min_p[r] * p[0]
            if top_k[r] > 0:
                keep[int(top_k[r]):] = False
            if top_p[r] < 1:
                keep &= p.cumsum(0) - p < top_p[r]
            keep &= x[order] > -math.inf
            keep[0] = True
            kept = order[keep]
            u = noise[r].double()[kept].clamp(torch.finfo(torch.float32).tiny, 1 - 2. ** -24)
            score = (x[kept] - x.max()) / temperature[r] - torch.log(-torch.log(u))
            token = int(kept[score.argmax()])
        tokens.append(token)
        logprobs.append(float(x[token] - torch.logsumexp(x, -1)))
    return torch.tensor(tokens), torch.tensor(logprobs, dtype=torch.float64)
