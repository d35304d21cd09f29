"""Measured cases of the serving operators: paged caches, attention over them, sampling.

A case is one pass through one operator, as a program that serves a language model calls it:

* ``kind='attn'``    ``paged_attn``: dense causal attention of a chunk of new tokens over a paged cache,
* ``kind='simp'``    ``paged_two_simplicial_attn``: the sliding-window 2-simplicial form,
* ``kind='append'``  ``paged_append``: keys and values of new tokens into the pages of one layer,
* ``kind='copy'``    ``copy_pages``: pages of every layer's pools to other pages (forks, compaction),
* ``kind='sample'``  ``sample_tokens``: next tokens from logits and given random numbers.

Ranges that the listed cases stand for (``draw`` samples them): 1 .. 64 sequences, 1 .. 2048 new tokens, caches of 1 .. 32768 tokens, 1 .. 16 heads
with 1 .. 8 query heads per key/value head, head dimensions 32 .. 256 (native and other ones), first windows 16 .. 1024, second windows 2 .. 64,
pages of 1 .. 128 tokens, bfloat16 (mostly) and float16; vocabularies of 256 .. 131072, float32 logits too.
"""
import math

import torch

own = False

_DTYPES = {'bf16': torch.bfloat16, 'fp16': torch.float16, 'fp32': torch.float32}


def _attn(name, b, n, h, hk, d, length, page, dtype='bf16', ragged=False):
    return {'name': name, 'kind': 'attn', 'b': b, 'n': n, 'h': h, 'hk': hk, 'd': d, 'length': length, 'page': page, 'dtype': dtype, 'ragged': ragged}


def _simp(name, b, n, h, hk, d, w1, w2, length, page, dtype='bf16', ragged=False):
    return {'name': name, 'kind': 'simp', 'b': b, 'n': n, 'h': h, 'hk': hk, 'd': d, 'w1': w1, 'w2': w2, 'length': length, 'page': page, 'dtype': dtype,
            'ragged': ragged}


def _append(name, b, n, sets, hk, d, length, page, dtype='bf16', ragged=False):
    return {'name': name, 'kind': 'append', 'b': b, 'n': n, 'sets': sets, 'hk': hk, 'd': d, 'length': length, 'page': page, 'dtype': dtype, 'ragged': ragged}


def _copy(name, pools, pages, pairs, hk, d, page, dtype='bf16'):
    return {'name': name, 'kind': 'copy', 'pools': pools, 'pages': pages, 'pairs': pairs, 'hk': hk, 'd': d, 'page': page, 'dtype': dtype}


def _sample(name, rows, vocab, dtype, filters):
    return {'name': name, 'kind': 'sample', 'rows': rows, 'vocab': vocab, 'dtype': dtype, 'filters': filters}


def listed():
    return [
        # the smallest call: one sequence, one new token, the language model's dense layer (latency and launches)
        _attn('attn_decode_smallest', 1, 1, 8, 4, 64, 300, 16),
        # a batch of conversations of different lengths, one new token each: all of the cache is read
        _attn('attn_decode_b16_l32768', 16, 1, 16, 4, 128, 32768, 64, ragged=True),
        # prefill: a chunk of a long document behind what is cached of it, at the long-context heads
        _attn('attn_chunk_n2048_l32768', 1, 2048, 16, 16, 128, 32768, 64),
        # one sequence, one new token, the simplicial layer of the language model
        _simp('simp_decode_smallest', 1, 1, 8, 4, 64, 512, 32, 700, 16),
        # short chunks of several sequences, none as long as another, a head dimension and windows off the native sizes
        _simp('simp_chunk_ragged_fp16_d96', 5, 77, 6, 2, 96, 300, 20, 2999, 24, 'fp16', True),
        # prefill of four documents at the headline heads and windows
        _simp('simp_chunk_b4_n1024_d128', 4, 1024, 8, 8, 128, 512, 32, 8192, 64),
        # a decode step of a full batch: one token of each sequence, both sets of a simplicial layer
        _append('append_decode_b64', 64, 1, 2, 4, 64, 2048, 16, ragged=True),
        # prefill of a training-sized batch, a dense layer
        _append('append_chunk_b8_n2048', 8, 2048, 1, 8, 64, 2048, 64),
        # eight samples forked from one prompt: the last, partly filled page of each, in all pools of the 12-layer model
        _copy('copy_fork_8', 36, 64, 8, 8, 64, 32),
        # compaction of a fragmented cache of that model
        _copy('copy_compact_512', 36, 1200, 512, 8, 64, 32),
        # byte-level model: 256 tokens, a few rows (latency)
        _sample('sample_bytes_8', 8, 256, 'fp32', True),
        # a large vocabulary, a full batch, every row with filters of its own
        _sample('sample_b96_v100000', 96, 100000, 'bf16', True),
    ]


# ---- geometry that a case fixes (the same for every seed)

def _lengths(c):
    """Tokens of each sequence in the cache, the new ones included."""
    if not c['ragged']:
        return [c['length']] * c['b']
    low = max(1, c['length'] // 8)
    return [c['length'] - (c['length'] - low) * ((i * 7) % c['b']) // max(1, c['b'] - 1) for i in range(c['b'])]


def _counts(c):
    """New tokens of each sequence; the other rows of the chunk are padding."""
    lengths = _lengths(c)
    if not c['ragged']:
        return [min(c['n'], length) for length in lengths]
    return [min(length, max(1, c['n'] - (c['n'] * i) // (2 * c['b']))) for i, length in enumerate(lengths)]


def _ramp(first, count, most):
    """sum over the positions first .. first + count - 1 of min(position + 1, most)"""
    below = max(0, min(count, most - first))
    return below * (2 * first + below + 1) // 2 + (count - below) * most


def _triples(first, count, w1, w2):
    return sum(min(p + 1, w1) * min(p + 1, w2) for p in range(first, first + count))


def work(case):
    """Inputs read once, outputs written once; two products for each attended key (pair of keys)."""
    c = case
    size = 4 if c['dtype'] == 'fp32' else 2
    if c['kind'] in ('attn', 'simp'):
        flops = moved = 0
        for length, count in zip(_lengths(c), _counts(c)):
            first = length - count
            moved += 2 * count * c['h'] * c['d'] * size
            if c['kind'] == 'attn':
                flops += 4 * c['d'] * c['h'] * _ramp(first, count, length)
                moved += 2 * length * c['hk'] * c['d'] * size
            else:
                flops += 4 * c['d'] * c['h'] * _triples(first, count, c['w1'], c['w2'])
                moved += 2 * (min(length, c['w1'] + count - 1) + min(length, c['w2'] + count - 1)) * c['hk'] * c['d'] * size
        return {'bytes': moved, 'flops': flops}
    if c['kind'] == 'append':
        return {'bytes': 2 * sum(_counts(c)) * 2 * c['sets'] * c['hk'] * c['d'] * size, 'flops': 0}
    if c['kind'] == 'copy':
        return {'bytes': 2 * c['pairs'] * c['pools'] * c['page'] * c['hk'] * c['d'] * size, 'flops': 0}
    # (random numbers are read where a token can win: everywhere without filters, at few tokens with them)
    each = size + (0 if c['filters'] else 4)
    return {'bytes': c['rows'] * (c['vocab'] * each + 12), 'flops': 0}


# ---- inputs

def prepare(case, seed):
    """Unit-variance q, k and v (what the per-head norms hand over) in pages that lie in the pool in no order; unused rows of the pages hold
    whatever was there before."""
    c = case
    g = torch.Generator(device='cuda').manual_seed(int(seed))
    dtype = _DTYPES[c['dtype']]
    randn = lambda *shape: torch.randn(*shape, generator=g, device='cuda').to(dtype)
    if c['kind'] == 'sample':
        rows = c['rows']
        rand = lambda: torch.rand(rows, generator=g, device='cuda')
        # peaked rows and flat ones
        logits = torch.randn(rows, c['vocab'], generator=g, device='cuda') * (1 + 2 * rand())[:, None]
        state = {'case': c, 'logits': logits.to(dtype), 'noise': torch.rand(rows, c['vocab'], generator=g, device='cuda')}
        state['temperature'] = (0.5 + rand()) * (rand() > 0.1)                     # (some rows are greedy)
        if c['filters']:
            state['top_k'] = (torch.rand(rows, generator=g, device='cuda') * 100).to(torch.int32)      # (0: off)
            state['top_p'], state['min_p'] = 0.5 + 0.6 * rand(), 0.1 * rand() * (rand() > 0.5)
        else:
            state['top_k'], state['top_p'], state['min_p'] = 0, 1., 0.
        return state
    if c['kind'] == 'copy':
        order = torch.randperm(c['pages'], generator=g, device='cuda').to(torch.int32).cpu()
        pairs = torch.stack([order[:c['pairs']], order[c['pairs']:2 * c['pairs']]], 1).contiguous()
        pools = randn(c['pools'], c['pages'], c['page'], c['hk'], c['d'])
        return {'case': c, 'pools': pools, 'each': pools.unbind(0), 'pairs': pairs}
    lengths, counts = _lengths(c), _counts(c)
    width = -(-max(lengths) // c['page'])
    pages = c['b'] * width + 3
    tables = torch.randperm(pages, generator=g, device='cuda')[:c['b'] * width].view(c['b'], width).to(torch.int32)
    state = {'case': c, 'tables': tables, 'most': max(lengths),
             'lengths': torch.tensor(lengths, dtype=torch.int32, device='cuda'), 'counts': torch.tensor(counts, dtype=torch.int32, device='cuda')}
    sets = {'attn': 1, 'simp': 2, 'append': c.get('sets')}[c['kind']]
    state['pages'] = [randn(pages, c['page'], c['hk'], c['d']) for _ in range(2 * sets)]      # keys first, then values
    if c['kind'] == 'append':
        state['rows'] = [randn(c['b'], c['n'], c['hk'], c['d']) for _ in range(2 * sets)]
    else:
        state['q'] = randn(c['b'], c['n'], c['h'], c['d'])
    return state


# ---- the operators as elementary operations, in 32 bits

def _positions(s):
    """(b, n) position of every row of the chunk, and whether it is a row at all"""
    n = s['case']['n']
    t = torch.arange(n, device='cuda')
    at = s['lengths'].long()[:, None] - s['counts'].long()[:, None] + t
    return at, (t < s['counts'][:, None]) & (at >= 0)


def _rows_at(s, pool, at):
    """Rows of a pool at positions ``at`` (b, ...): (b, ..., hk, d) in 32 bits; positions below 0 read some row"""
    page = s['case']['page']
    flat = at.clamp(0, s['tables'].shape[1] * page - 1).flatten(1)
    index = s['tables'].long().gather(1, flat // page) * page + flat % page
    return pool.flatten(0, 1)[index].float().unflatten(1, at.shape[1:])


def _softmax_weights(logits, mask):
    logits = logits.masked_fill(~mask, -math.inf)
    top = logits.amax(-1, keepdim=True)
    weights = (logits - top.masked_fill(top == -math.inf, 0.)).exp()
    return weights / weights.sum(-1, keepdim=True).clamp(min=1e-30)


def _plain_attn(s):
    c = s['case']
    at, real = _positions(s)
    keys = torch.arange(s['most'], device='cuda').expand(c['b'], -1)
    k, v = (_rows_at(s, pool, keys).permute(0, 2, 1, 3) for pool in s['pages'])                       # b hk L d
    q = s['q'].float().unflatten(2, (c['hk'], -1)).permute(0, 2, 3, 1, 4).flatten(2, 3)               # b hk (g n) d
    group = c['h'] // c['hk']
    mask = ((keys[:, None, :] <= at[:, :, None]) & real[:, :, None])[:, None].repeat(1, 1, group, 1)  # b 1 (g n) L
    weights = _softmax_weights(torch.matmul(q, k.transpose(-1, -2).contiguous()) * c['d'] ** -0.5, mask)
    out = torch.matmul(weights, v.contiguous()).unflatten(2, (group, c['n']))
    return out.permute(0, 3, 1, 2, 4).flatten(2, 3).to(s['q'].dtype)


def _plain_simp(s):
    c = s['case']
    at, real = _positions(s)
    j1, j2 = (at[:, :, None] - torch.arange(w, device='cuda') for w in (c['w1'], c['w2']))            # b n w
    k1, k2, v1, v2 = (_rows_at(s, pool, j).permute(0, 3, 1, 2, 4) for pool, j in zip(s['pages'], (j1, j2, j1, j2)))      # b hk n w d
    q = s['q'].float().unflatten(2, (c['hk'], -1)).permute(0, 2, 1, 3, 4)                             # b hk n g d
    a = (q[:, :, :, :, None] * k2[:, :, :, None]).flatten(3, 4)                                       # b hk n (g w2) d
    logits = torch.matmul(a, k1.transpose(-1, -2).contiguous()).unflatten(3, (-1, c['w2'])) * c['d'] ** -0.5
    mask = ((j2 >= 0)[:, :, :, None] & (j1 >= 0)[:, :, None] & real[:, :, None, None])[:, None, :, None]      # b 1 n 1 w2 w1
    weights = _softmax_weights(logits.flatten(4), mask.expand_as(logits).flatten(4)).view_as(logits)
    mixed = torch.matmul(weights.flatten(3, 4), v1.contiguous()).unflatten(3, (-1, c['w2']))          # b hk n g w2 d
    out = (mixed * v2[:, :, :, None]).sum(4)
    return out.permute(0, 2, 1, 3, 4).flatten(2, 3).to(s['q'].dtype)


def _plain_append(s):
    c = s['case']
    at, real = _positions(s)
    flat = at.clamp(min=0)
    index = (s['tables'].long().gather(1, flat // c['page'] % s['tables'].shape[1]) * c['page'] + flat % c['page'])[real]
    return [pool.flatten(0, 1).index_copy_(0, index, rows[real]).view_as(pool) for pool, rows in zip(s['pages'], s['rows'])]


def _plain_copy(s):
    src, dst = s['pairs'].long().cuda().unbind(1)
    s['pools'][:, dst] = s['pools'][:, src]
    return s['pools']


def _column(v):
    return v[:, None] if torch.is_tensor(v) else v


def _plain_sample(s):
    x = s['logits'].float().nan_to_num(nan=-math.inf, posinf=torch.finfo(torch.float32).max, neginf=-math.inf)
    xs, index = x.sort(dim=-1, descending=True, stable=True)
    t = s['temperature'][:, None]
    greedy = t <= 0
    scaled = (xs - xs[:, :1]) / torch.where(greedy, 1., t)
    weights = scaled.exp()
    mass, top_k, top_p, min_p = weights.cumsum(-1), _column(s['top_k']), _column(s['top_p']), _column(s['min_p'])
    rank = torch.arange(x.shape[1], device='cuda')
    kept = ((rank < top_k) | (top_k <= 0)) & ((mass - weights < top_p * mass[:, -1:]) | (top_p >= 1)) & (weights >= min_p)
    kept = (kept & ~greedy) | (rank == 0)
    tiny, most = torch.finfo(torch.float32).tiny, 1 - 2. ** -24
    score = scaled - (-s['noise'].gather(1, index).clamp(tiny, most).log()).log()
    best = score.masked_fill(~kept, -math.inf).argmax(-1, keepdim=True)
    chosen = xs.gather(1, best) - xs[:, :1] - (xs - xs[:, :1]).exp().sum(-1, keepdim=True).log()
    return index.gather(1, best)[:, 0], chosen[:, 0]


def run(state):
    c, s = state['case'], state
    if not own:
        return {'attn': _plain_attn, 'simp': _plain_simp, 'append': _plain_append, 'copy': _plain_copy, 'sample': _plain_sample}[c['kind']](s)
    import simplicial_attention_amd as sa
    if c['kind'] == 'attn':
        return sa.paged_attn(s['q'], *s['pages'], s['tables'], s['lengths'], s['counts'], max_length=s['most'])
    if c['kind'] == 'simp':
        return sa.paged_two_simplicial_attn(s['q'], s['pages'][:2], s['pages'][2:], s['tables'], s['lengths'], s['counts'], w1=c['w1'], w2=c['w2'])
    if c['kind'] == 'append':
        sa.paged_append(s['pages'], s['rows'], s['tables'], s['lengths'], s['counts'])
        return list(s['pages'])
    if c['kind'] == 'copy':
        sa.copy_pages(s['each'], s['pairs'])
        return s['pools']
    return sa.sample_tokens(s['logits'], s['noise'], temperature=s['temperature'], top_k=s['top_k'], top_p=s['top_p'], min_p=s['min_p'])


# ---- the same from the definition, in 64 bits, sequence by sequence

def exact(case, seed):
    c = case
    s = prepare(case, seed)
    if c['kind'] == 'copy':
        pools = s['pools'].double()
        for src, dst in s['pairs'].tolist():
            pools[:, dst] = s['pools'][:, src].double()
        return pools
    if c['kind'] == 'sample':
        return _exact_sample(s)
    lengths, counts = _lengths(c), _counts(c)
    ps = c['page']
    if c['kind'] == 'append':
        pools = [p.double() for p in s['pages']]
        for i, (length, count) in enumerate(zip(lengths, counts)):
            position = torch.arange(length - count, length, device='cuda')
            page, row = s['tables'][i].long()[position // ps], position % ps
            for pool, rows in zip(pools, s['rows']):
                pool[page, row] = rows[i, :count].double()
        return pools
    out = torch.zeros(s['q'].shape, dtype=torch.float64, device='cuda')
    group = c['h'] // c['hk']
    for i, (length, count) in enumerate(zip(lengths, counts)):
        whole = [p[s['tables'][i].long()].flatten(0, 1)[:length].double() for p in s['pages']]         # L hk d
        first = length - count
        for head in range(c['h']):
            q = s['q'][i, :count, head].double() / math.sqrt(c['d'])
            t = [p[:, head // group] for p in whole]
            if c['kind'] == 'attn':
                logits = q @ t[0].T
                future = torch.arange(length, device='cuda') > torch.arange(first, length, device='cuda')[:, None]
                out[i, :count, head] = torch.softmax(logits.masked_fill_(future, -math.inf), -1) @ t[1]
                continue
            k1, k2, v1, v2 = t
            for lo in range(0, count, 256):
                at = torch.arange(first + lo, first + min(count, lo + 256), device='cuda')
                a, b = at[:, None] - torch.arange(c['w1'], device='cuda'), at[:, None] - torch.arange(c['w2'], device='cuda')
                pair = torch.bmm(q[lo:lo + 256, None] * k2[b.clamp(min=0)], k1[a.clamp(min=0)].mT.contiguous())       # rows w2 w1
                pair.masked_fill_((a < 0)[:, None] | (b < 0)[:, :, None], -math.inf)
                p = torch.softmax(pair.flatten(1), -1).view_as(pair)
                out[i, lo:lo + 256, head][:len(at)] = (torch.bmm(p, v1[a.clamp(min=0)]) * v2[b.clamp(min=0)]).sum(1)
    return out


def _exact_sample(s):
    tokens, chosen = [], []
    for i in range(s['case']['rows']):
        x = s['logits'][i].double()
        order = sorted_order = torch.sort(x, descending=True, stable=True).indices
        t = float(s['temperature'][i])
        if t > 0:
            p = torch.softmax(x / t, -1)[sorted_order]
            k, top_p, min_p = (float(s[name][i]) if torch.is_tensor(s[name]) else s[name] for name in ('top_k', 'top_p', 'min_p'))
            keep = p >= min_p * p[0]
            if k > 0:
                keep[int(k):] = False
            if top_p < 1:
                keep &= p.cumsum(0) - p < top_p
            keep[0] = True
            order = sorted_order[keep]
            u = s['noise'][i].double()[order].clamp(torch.finfo(torch.float32).tiny, 1 - 2. ** -24)
            token = int(order[(x[order] / t - torch.log(-torch.log(u))).argmax()])
        else:
            token = int(order[0])
        tokens.append(token)
        chosen.append(float(x[token] - torch.logsumexp(x, -1)))
    return torch.tensor(tokens, device='cuda'), torch.tensor(chosen, dtype=torch.float64, device='cuda')


# ---- more cases of the same ranges

# a drawn case costs at most what the largest listed one of its kind does
_MOST_FLOPS = {'attn': work(listed()[2])['flops'], 'simp': work(listed()[5])['flops']}
_MOST_BYTES = {'attn': work(listed()[1])['bytes'], 'simp': 1 << 30, 'append': 1 << 28, 'copy': work(listed()[9])['bytes'], 'sample': 96 * 100000 * 6}
_MOST_LOGITS = {'attn': 16 * 2048 * 32768, 'simp': 4 * 8 * 1024 * 512 * 32}
_MOST_GATHERED = 4 * 8 * 1024 * 512 * 128


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _fits(c):
    w = work(c)
    if w['bytes'] > _MOST_BYTES[c['kind']] or w['flops'] > _MOST_FLOPS.get(c['kind'], 0):
        return False
    if c['kind'] == 'attn':
        return c['b'] * c['h'] * c['n'] * c['length'] <= _MOST_LOGITS['attn'] and c['b'] * c['length'] * c['hk'] * c['d'] <= 16 * 32768 * 4 * 128
    if c['kind'] == 'simp':
        return (c['b'] * c['n'] * c['h'] * c['w1'] * c['w2'] <= _MOST_LOGITS['simp'] and c['b'] * c['n'] * c['hk'] * c['w1'] * c['d'] <= _MOST_GATHERED
                and c['b'] * c['length'] * c['hk'] * c['d'] * 8 <= 1 << 31)
    return True


def draw(rng):
    while True:
        kind = rng.choice(['attn', 'attn', 'attn', 'simp', 'simp', 'simp', 'append', 'copy', 'sample', 'sample'])
        hk = rng.choice([1, 2, 4, 8])
        h = hk * rng.choice([g for g in (1, 2, 4, 8) if hk * g <= 16])
        d = rng.choice([32, 64, 64, 64, 128, 128, 128, 256, 48, 80, 96])
        dtype, page, b = rng.choice(['bf16'] * 3 + ['fp16']), rng.choice([1, 8, 16, 16, 24, 32, 64, 128]), _log_uniform(rng, 1, 64)
        n = rng.choice([1, _log_uniform(rng, 2, 16), _log_uniform(rng, 17, 2048)])
        ragged = rng.random() < 0.5
        if kind == 'attn':
            case = _attn('', b, n, h, hk, d, max(n, _log_uniform(rng, 1, 32768)), page, dtype, ragged)
        elif kind == 'simp':
            case = _simp('', b, n, h, hk, d, _log_uniform(rng, 16, 1024), _log_uniform(rng, 2, 64), max(n, _log_uniform(rng, 1, 8192)), page, dtype, ragged)
        elif kind == 'append':
            case = _append('', b, n, rng.choice([1, 2]), hk, d, max(n, _log_uniform(rng, 1, 8192)), page, dtype, ragged)
            if case['b'] * case['length'] * hk * d * case['sets'] > 1 << 28:
                continue
        elif kind == 'copy':
            pairs = _log_uniform(rng, 1, 512)
            case = _copy('', rng.randint(2, 48), 2 * pairs + rng.randint(1, 64), pairs, hk, d, page, dtype)
        else:
            case = _sample('', _log_uniform(rng, 1, 256), _log_uniform(rng, 256, 131072), rng.choice(['bf16', 'fp16', 'fp32']), rng.random() < 0.6)
        del case['name']
        if _fits(case):
            return case
