"""Paged caches: attention of new tokens over them (dense and 2-simplicial), rows into pages, pages to pages."""
import pytest
import torch

import simplicial_attention_amd as S
from simplicial_attention_amd import _native
from tests import paged_util as P

pytestmark = pytest.mark.gpu
BF16, F16 = torch.bfloat16, torch.float16
NAN, INF = float('nan'), float('inf')


def ints(*values):
    return torch.tensor(values, dtype=torch.int32, device='cuda')


def queries(b, n, h, d, dtype=BF16, seed=7, std=1.):
    return (torch.randn(b, n, h, d, generator=torch.Generator().manual_seed(seed)) * std).to(dtype).cuda()


def run(q, pools, tables, lengths, counts=None, **kw):
    if len(pools) == 2:
        return S.paged_attn(q, *pools, tables, lengths, counts, **kw)
    return S.paged_two_simplicial_attn(q, pools[:2], pools[2:], tables, lengths, counts, **kw)


def want(q, pools, tables, lengths, counts=None, **kw):
    half = len(pools) // 2
    return P.attend(q, pools[:half], pools[half:], tables, lengths, counts, **kw)


# b, n, h, hk, d, lengths, page, dtype
DENSE = [
    (1, 1, 8, 4, 64, [300], 16, BF16),                 # one token
    (1, 1, 1, 1, 64, [1], 16, BF16),                   # of a sequence of one
    (3, 1, 4, 2, 128, [1, 33, 2500], 16, BF16),        # keys beyond one LDS segment, shared out
    (2, 1, 16, 2, 32, [31, 32], 1, F16),               # pages of one row
    (2, 1, 8, 8, 256, [500, 65], 24, BF16),
    (2, 3, 4, 1, 64, [64, 100], 8, BF16),              # a few tokens, all heads on one key/value head
    (2, 8, 4, 1, 128, [8, 40], 64, F16),               # rows fill the 32 columns exactly
    (2, 9, 4, 1, 64, [9, 77], 16, BF16),               # one more than that
    (1, 40, 6, 2, 96, [333], 24, F16),                 # padded head dimension
    (2, 70, 2, 1, 48, [70, 129], 128, BF16),
    (1, 130, 3, 3, 40, [700], 7, BF16),                # rows of 80 bytes, odd pages
    (1, 65, 4, 4, 128, [2200], 32, BF16),
    (1, 37, 2, 2, 256, [90], 16, F16),
    (5, 33, 2, 2, 32, [33, 64, 65, 96, 200], 16, BF16),
]


@pytest.mark.parametrize('case', DENSE, ids=lambda c: '-'.join(map(str, c[:5])) + f'-p{c[6]}')
def test_dense(case):
    b, n, h, hk, d, lengths, page, dtype = case
    pools, tables = P.make_cache(b, hk, d, lengths, page, 1, dtype)
    q = queries(b, n, h, d, dtype)
    P.check(run(q, pools, tables, ints(*lengths)), want(q, pools, tables, lengths))


# ... w1, w2
SIMPLICIAL = [
    (1, 1, 8, 4, 64, [700], 16, BF16, 512, 32),
    (1, 1, 2, 1, 64, [1], 16, BF16, 512, 32),
    (3, 1, 4, 2, 128, [5, 40, 600], 16, BF16, 100, 7),
    (2, 2, 2, 2, 32, [20, 90], 1, F16, 33, 33),        # a second block of offsets with one offset
    (2, 1, 2, 1, 256, [70, 300], 24, BF16, 64, 32),
    (1, 3, 2, 2, 64, [200], 16, BF16, 128, 70),        # three blocks of offsets
    (1, 1, 2, 1, 64, [3000], 64, BF16, 2500, 2),       # a first window beyond one LDS segment
    (1, 5, 2, 1, 64, [50], 16, BF16, 1, 1),            # windows of one
    (2, 20, 2, 2, 64, [20, 300], 16, BF16, 50, 32),
    (2, 19, 6, 2, 96, [19, 333], 24, F16, 90, 20),
    (1, 40, 4, 1, 128, [100], 8, BF16, 64, 40),
    (1, 21, 2, 2, 256, [60], 16, BF16, 40, 16),
    (1, 33, 3, 3, 40, [300], 7, F16, 200, 9),
    (2, 17, 2, 1, 32, [17, 64], 64, BF16, 512, 64),
]


@pytest.mark.parametrize('case', SIMPLICIAL, ids=lambda c: '-'.join(map(str, c[:5])) + f'-w{c[8]}-{c[9]}')
def test_simplicial(case):
    b, n, h, hk, d, lengths, page, dtype, w1, w2 = case
    pools, tables = P.make_cache(b, hk, d, lengths, page, 2, dtype)
    q = queries(b, n, h, d, dtype)
    P.check(run(q, pools, tables, ints(*lengths), w1=w1, w2=w2), want(q, pools, tables, lengths, w1=w1, w2=w2))


# batch, new tokens, h, hk, d, page, lengths (a number: drawn up to it), dtype
UNEVEN = [
    (4, 70, 4, 2, 64, 16, [3000, 0, 40, 70], BF16),
    (3, 33, 2, 1, 256, 64, [1, 2500, 900], BF16),
    (5, 50, 2, 2, 128, 24, [33, 2000, 50, 1999, 700], F16),
    (64, 40, 1, 1, 32, 16, 1500, BF16),
    (65, 40, 1, 1, 32, 16, 600, BF16),                  # more sequences than a wave has lanes: even shares
    (2, 300, 8, 1, 64, 32, [6000, 350], BF16),
]


@pytest.mark.parametrize('case', UNEVEN, ids=lambda c: '-'.join(map(str, c[:5])))
def test_shares_of_sequences_of_different_lengths(case):
    b, n, h, hk, d, page, lengths, dtype = case
    if isinstance(lengths, int):
        lengths = torch.randint(0, lengths + 1, (b,), generator=torch.Generator().manual_seed(3)).tolist()
    counts = [min(n, x) if i % 3 else n for i, x in enumerate(lengths)]
    pools, tables = P.make_cache(b, hk, d, lengths, page, 1, dtype)
    q = queries(b, n, h, d, dtype)
    out = run(q, pools, tables, ints(*lengths), ints(*counts))
    P.check(out, want(q, pools, tables, lengths, counts))
    # the same bits again, and nothing but rounding where a sequence is alone
    assert torch.equal(out, run(q, pools, tables, ints(*lengths), ints(*counts)))
    alone = torch.cat([run(q[i:i + 1], pools, tables[i:i + 1], ints(lengths[i]), ints(counts[i])) for i in range(b)])
    P.check(alone, want(q, pools, tables, lengths, counts))


@pytest.mark.parametrize('w2', [1, 2, 3, 4, 7, 8, 9, 16])
@pytest.mark.parametrize('d,g', [(32, 4), (64, 3), (104, 2), (256, 2)])
def test_short_second_windows_of_many_tokens(w2, d, g):
    """Several (token, head) units of a wave: ends of sequences, rows and tokens that are not there, heads of a group, first windows that differ by unit."""
    b, n, hk, lengths = 3, 131, 2, [131, 40, 390]
    counts = [131, 57, 100]
    pools, tables = P.make_cache(b, hk, d, lengths, 16, 2, BF16)
    q = queries(b, n, hk * g, d)
    for w1 in (33, 300):
        out = run(q, pools, tables, ints(*lengths), ints(*counts), w1=w1, w2=w2)
        P.check(out, want(q, pools, tables, lengths, counts, w1=w1, w2=w2))


@pytest.mark.parametrize('n', [64, 65, 100, 128, 129, 140])
def test_short_second_windows_on_either_side_of_the_rule(n):
    """512, 520, 800, 1024, 1032 and 1120 (token, head) units."""
    pools, tables = P.make_cache(2, 1, 32, [n + 20, n], 16, 2, BF16)
    q = queries(2, n, 4, 32)
    P.check(run(q, pools, tables, ints(n + 20, n), w1=40, w2=8), want(q, pools, tables, [n + 20, n], w1=40, w2=8))


@pytest.mark.parametrize('bad', [float('nan'), float('inf'), -float('inf')])
def test_units_of_a_wave_keep_their_windows(bad):
    """Short second windows: a row that is no number reaches the units whose first or second window holds it, and not their neighbours in the wave."""
    n, at = 150, 77
    pools, tables = P.make_cache(2, 1, 64, [n, n], 16, 2, BF16)
    q = queries(2, n, 4, 64)
    for pool in pools:
        for s in range(2):
            pool[tables[s, (at + s) // 16].long(), (at + s) % 16] = bad
        out = run(q, pools, tables, ints(n, n), w1=20, w2=4)
        touched = torch.zeros(2, n, dtype=torch.bool, device='cuda')
        for s in range(2):
            touched[s, at + s:at + s + 20] = True
        clean = P.make_cache(2, 1, 64, [n, n], 16, 2, BF16)[0]
        expected = want(q, clean, tables, [n, n], w1=20, w2=4)
        P.check(out[~touched], expected[~touched])


def test_short_second_window_in_shares():
    """... where the keys of few units are split, and joined."""
    pools, tables = P.make_cache(1, 1, 64, [9000], 64, 2, F16)
    q = queries(1, 1100, 1, 64, F16)
    P.check(run(q, pools, tables, ints(9000), w1=8000, w2=5), want(q, pools, tables, [9000], w1=8000, w2=5))


@pytest.mark.parametrize('n', [1, 6, 45])
@pytest.mark.parametrize('sets', [1, 2])
def test_rows_that_are_not_there(n, sets):
    """Padding, sequences of no tokens, more rows than tokens: zeros, and the others as ever."""
    b, lengths = 6, [0, 3, 50, 80, 2, 64]
    counts = [0, min(n, 3), 0, n, n + 5, max(n - 2, -3)]
    pools, tables = P.make_cache(b, 2, 64, lengths, 16, sets)
    q = queries(b, n, 4, 64)
    kw = dict(w1=40, w2=12) if sets == 2 else {}
    out = run(q, pools, tables, ints(*lengths), ints(*counts), **kw)
    P.check(out, want(q, pools, tables, lengths, counts, **kw))
    assert not out[0].any() and not out[2].any()


@pytest.mark.parametrize('n', [1, 7, 50])
@pytest.mark.parametrize('sets', [1, 2])
def test_places_that_are_not_there(n, sets):
    """Missing pages (entries of any value) and lengths beyond the table."""
    b, lengths = 3, [100, 100, 104]
    pools, tables = P.make_cache(b, 1, 64, lengths, 8, sets, garbage=1e30)
    tables[0, 3], tables[0, 12], tables[1, :] = -1, 2 ** 31 - 1, -7
    tables[2, 5:7] = pools[0].shape[0]
    long = [100, 100, 120]                   # (the table of the third reaches 104)
    q = queries(b, n, 2, 64)
    kw = dict(w1=60, w2=20) if sets == 2 else {}
    out = run(q, pools, tables, ints(*long), **kw)
    P.check(out, want(q, pools, tables, long, **kw))
    assert not out[1].any()


@pytest.mark.parametrize('bad', [NAN, INF])
@pytest.mark.parametrize('n', [4, 50])
@pytest.mark.parametrize('sets', [1, 2])
def test_values_of_masked_keys_reach_no_row(sets, n, bad):
    """A key or value that is not a number touches the rows that attend it and no other: new tokens in front of it, windows behind it."""
    length = 120
    pools, tables = P.make_cache(1, 1, 64, [length], 16, sets, seed=3)
    q = queries(1, n, 2, 64)
    kw = dict(w1=30, w2=6) if sets == 2 else {}
    at = length - n // 2                     # the position of a new token
    for pool in (pools[0], pools[-1]) if sets == 1 else pools:
        pool[int(tables[0, at // 16]), at % 16, 0, 5::16] = bad
    if sets == 2:                            # and one that only the first row's window holds
        old = length - n - 29
        pools[2][int(tables[0, old // 16]), old % 16] = bad
    out = run(q, pools, tables, ints(length), **kw)
    reference = want(q, pools, tables, [length], **kw)
    finite = torch.isfinite(reference).all(-1)
    assert torch.isfinite(out).all(-1).equal(finite)
    assert finite.any() and not finite.all()
    P.check(out[finite], reference[finite])


@pytest.mark.parametrize('dtype', [BF16, F16])
@pytest.mark.parametrize('n', [1, 40])
@pytest.mark.parametrize('sets', [1, 2])
def test_logits_that_grow_along_the_keys(sets, n, dtype):
    """Later keys outweigh earlier ones by far more than the reference of the softmax allows for, and the other way round."""
    length, page = 400, 16
    for falling in (False, True):
        pools, tables = P.make_cache(1, 1, 64, [length], page, sets, dtype, seed=5, std=0.3)
        x = torch.arange(length, device='cuda')
        growth = (x.flip(0) if falling else x).float() / length * 20
        k1 = pools[0]
        k1[tables[0].long()[x // page], x % page, 0, 0] = growth.to(dtype)
        q = queries(1, n, 2, 64, dtype, std=0.3)
        q[..., 0] = 40
        kw = dict(w1=300, w2=8) if sets == 2 else {}
        if sets == 2:
            pools[1][..., 0] = 1
        P.check(run(q, pools, tables, ints(length), **kw), want(q, pools, tables, [length], **kw))


@pytest.mark.parametrize('sets', [1, 2])
def test_strides_and_other_streams(sets):
    """Pools that are slices of larger tensors, queries with heads in front, tables with a stride: on a stream of their own."""
    b, n, h, hk, d, page, lengths = 2, 5, 4, 2, 64, 16, [37, 90]
    pools, tables = P.make_cache(b, hk, d, lengths, page, sets)
    joint = torch.full((pools[0].shape[0], 2 * sets, page, hk + 1, d + 8), NAN, dtype=BF16, device='cuda')
    views = [joint[:, i, :, 1:, 8:] for i in range(2 * sets)]
    for view, pool in zip(views, pools):
        view.copy_(pool)
    wide = torch.full((b, 3 * tables.shape[1]), -1, dtype=torch.int32, device='cuda')
    wide[:, ::3] = tables
    q = queries(b, h, n, d + 3).transpose(1, 2)[..., 3:]
    kw = dict(w1=40, w2=12) if sets == 2 else {}
    reference = want(q, pools, tables, lengths, **kw)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        out = run(q, views, wide[:, ::3], ints(*lengths), **kw)
        column = wide[:, :1].clone()
    torch.cuda.current_stream().wait_stream(stream)
    P.check(out, reference)
    assert column.shape == (b, 1)


def test_pools_beyond_32_bits():
    """Pages whose offset in the pool passes 4 GiB."""
    page, hk, d, n = 64, 4, 64, 3
    pages = (5 << 30) // (page * hk * d * 2)
    pools = [torch.empty(pages, page, hk, d, dtype=BF16, device='cuda') for _ in range(4)]
    tables = ints(pages - 1, 5, pages - 7, pages // 2 + 3).view(1, 4)
    length = 4 * page - 9
    rows = [torch.randn(1, length, hk, d, device='cuda', dtype=BF16) for _ in range(4)]
    S.paged_append(pools, rows, tables, ints(length))
    small = [torch.zeros(4, page, hk, d, dtype=BF16, device='cuda') for _ in range(4)]
    for pool, r in zip(small, rows):
        pool.flatten(0, 1)[:length] = r[0]
    q, flat = queries(1, n, 4, d), ints(0, 1, 2, 3).view(1, 4)
    for width in (1, 40):
        qq = q if width == 1 else queries(1, width, 4, d)
        assert torch.equal(run(qq, pools[:2], tables, ints(length)), run(qq, small[:2], flat, ints(length)))
        assert torch.equal(run(qq, pools, tables, ints(length), w1=200, w2=16), run(qq, small, flat, ints(length), w1=200, w2=16))
    P.check(run(q, pools[:2], tables, ints(length)), want(q, small[:2], flat, [length]))
    S.copy_pages(pools, [(pages - 1, 3), (pages - 7, pages - 2)])
    for pool, r in zip(pools, rows):
        assert torch.equal(pool[3], r[0, :page]) and torch.equal(pool[pages - 2], r[0, 2 * page:3 * page])


@pytest.mark.parametrize('sets', [1, 2])
@pytest.mark.parametrize('hint', [None, 0, 10, 100000])
def test_max_length_is_only_a_hint(sets, hint):
    b, n, lengths = 2, 2, [3000, 257]
    pools, tables = P.make_cache(b, 1, 64, lengths, 16, sets)
    q = queries(b, n, 2, 64)
    kw = dict(w1=700, w2=9) if sets == 2 else {}
    P.check(run(q, pools, tables, ints(*lengths), max_length=hint, **kw), want(q, pools, tables, lengths, **kw))


@pytest.mark.parametrize('n', [1, 64])
def test_a_chunk_equals_its_tokens_one_by_one(n):
    """The same rows from one call and from single-token calls agree to the rounding of either."""
    length, page = 500, 16
    pools, tables = P.make_cache(1, 2, 64, [length], page, 2)
    q = queries(1, n, 4, 64)
    for kw, p in ((dict(), pools[:2]), (dict(w1=128, w2=32), pools)):
        whole = run(q, p, tables, ints(length), **kw)
        for t in range(0, n, 9):
            one = run(q[:, t:t + 1], p, tables, ints(length - n + 1 + t), **kw)
            P.check(one, whole[:, t:t + 1].double())


def test_results_do_not_change_from_call_to_call():
    pools, tables = P.make_cache(2, 2, 128, [3000, 1111], 16, 2)
    for n in (1, 70):
        q = queries(2, n, 4, 128)
        for p, kw in ((pools[:2], {}), (pools, dict(w1=512, w2=32))):
            first = run(q, p, tables, ints(3000, 1111), **kw)
            for _ in range(3):
                assert torch.equal(run(q, p, tables, ints(3000, 1111), **kw), first)


def test_agrees_with_the_training_kernels():
    """A whole sequence as one chunk: what sliding_two_simplicial_attn computes."""
    b, n, h, hk, d, page = 2, 150, 4, 2, 64, 16
    rows = [torch.randn(b, n, hk, d, device='cuda', dtype=BF16) for _ in range(4)]
    pools, tables = P.make_cache(b, hk, d, [n, n], page, 2)
    lengths = ints(n, n)
    S.paged_append(pools, rows, tables, lengths)
    q = queries(b, n, h, d)
    got = S.paged_two_simplicial_attn(q, pools[:2], pools[2:], tables, lengths, w1=64, w2=20)
    same = S.sliding_two_simplicial_attn(q, rows[:2], rows[2:], w1=64, w2=20)
    assert float((got.double() - same.double()).norm() / same.double().norm()) < 2 * P.NORM[BF16]


@pytest.mark.parametrize('source', [BF16, F16, torch.float32])
@pytest.mark.parametrize('target', [BF16, F16])
@pytest.mark.parametrize('d', [64, 40, 37])
def test_append(source, target, d):
    b, n, hk, page, dim = 4, 6, 2, 5, -(-d // 8) * 8
    lengths, counts = [6, 23, 2, 9], [6, 4, 5, 0]                     # (the third: rows before the sequence are not written)
    width = 6
    pages = b * width
    tables = torch.randperm(pages, generator=torch.Generator().manual_seed(1)).view(b, width).to(torch.int32).cuda()
    tables[1, 4] = -1                                                # positions 20 .. 22 of the second are not there
    pools = [torch.full((pages, page, hk, dim), 7., dtype=target, device='cuda') for _ in range(3)]
    rows = [torch.randn(b, n, hk, d, device='cuda').to(source) for _ in range(3)]
    expected = [p.clone() for p in pools]
    for s in range(b):
        for t in range(counts[s]):
            x = lengths[s] - counts[s] + t
            if x < 0 or int(tables[s, x // page]) < 0:
                continue
            for e, r in zip(expected, rows):
                e[int(tables[s, x // page]), x % page] = 0
                e[int(tables[s, x // page]), x % page, :, :d] = r[s, t].to(target)
    S.paged_append(pools, rows, tables, ints(*lengths), ints(*counts))
    for p, e in zip(pools, expected):
        assert torch.equal(p, e)


@pytest.mark.parametrize('pairs', [1, 7, 300])
@pytest.mark.parametrize('shape', [(4, 2, 64), (3, 1, 5), (24, 8, 128)])
def test_copy_pages(pairs, shape):
    pages = 2 * pairs + 5
    pools = [torch.randn(pages, *shape, device='cuda').to(t) for t in (BF16, F16, BF16)] + [torch.randn(pages, 3, 1, 2, device='cuda')]
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(pairs))
    moves = torch.stack([order[:pairs], order[pairs:2 * pairs]], 1)
    expected = [p.clone() for p in pools]
    for e in expected:
        e[moves[:, 1].cuda()] = e[moves[:, 0].cuda()]
    S.copy_pages(pools, moves)
    for p, e in zip(pools, expected):
        assert torch.equal(p, e)
    S.copy_pages(pools, [])
    many = [torch.randn(9, 2, 1, 8, device='cuda') for _ in range(70)]
    S.copy_pages(many, [(1, 2), (1, 3)])                             # one page may go to several
    assert all(torch.equal(p[1], p[2]) and torch.equal(p[1], p[3]) for p in many)


def test_refusals():
    pools, tables = P.make_cache(2, 2, 64, [20, 20], 16, 2)
    q, lengths = queries(2, 1, 4, 64), ints(20, 20)
    k, v = pools[:2]
    with pytest.raises(AssertionError):
        S.paged_attn(q.cpu(), k, v, tables, lengths)
    with pytest.raises(AssertionError):
        S.paged_two_simplicial_attn(q, (k,), (v, v), tables, lengths)
    with pytest.raises(TypeError):
        S.paged_attn(q.half(), k, v, tables, lengths)
    with pytest.raises(TypeError):
        S.paged_attn(q.float(), k.float(), v.float(), tables, lengths)
    with pytest.raises(TypeError):
        S.paged_attn(q, k, v, tables.long(), lengths)
    with pytest.raises(ValueError):
        S.paged_attn(q, k, v, tables, lengths[:1])
    with pytest.raises(ValueError):
        S.paged_attn(q, k, v, tables, lengths, ints(1, 1, 1))
    with pytest.raises(ValueError):
        S.paged_attn(q, k, v[:-1], tables, lengths)
    with pytest.raises(ValueError):
        S.paged_attn(queries(2, 1, 3, 64), k, v, tables, lengths)
    with pytest.raises(ValueError):
        S.paged_attn(q, k[..., ::2], v[..., ::2], tables, lengths)
    with pytest.raises(NotImplementedError):
        S.paged_attn(queries(2, 1, 4, 72), k, v, tables, lengths)
    with pytest.raises(NotImplementedError):
        S.paged_attn(q[..., :60], k[..., :60], v[..., :60], tables, lengths)
    with pytest.raises(ValueError):
        S.paged_two_simplicial_attn(q, pools[:2], pools[2:], tables, lengths, w1=0)
    with pytest.raises(ValueError):
        S.paged_attn(q, k, v, tables, lengths, max_length=-1)
    with pytest.raises(_native.Sa2Error):
        S.paged_attn(q, k, v, tables, lengths, scale=NAN)
    with pytest.raises(RuntimeError):
        S.paged_attn(q.requires_grad_(), k, v, tables, lengths)
    with torch.no_grad():
        S.paged_attn(q, k, v, tables, lengths)
    with pytest.raises(ValueError):
        S.paged_append([k, v], [q], tables, lengths)
    with pytest.raises(ValueError):
        S.paged_append([k], [queries(2, 1, 4, 64)], tables, lengths)
    with pytest.raises(TypeError):
        S.paged_append([k], [queries(2, 1, 2, 64).double()], tables, lengths)
    for pairs in ([(0, 1), (2, 1)], [(0, 1), (1, 2)], [(0, 0)], [(-1, 0)], [(0, k.shape[0])], torch.tensor([[0, 1 << 40]])):
        with pytest.raises((ValueError, _native.Sa2Error)):
            S.copy_pages([k, v], pairs)
    with pytest.raises(ValueError):
        S.copy_pages([k.transpose(1, 2)], [(0, 1)])
    with pytest.raises(ValueError):
        S.copy_pages([k], torch.tensor([[0, 1]], device='cuda'))


@pytest.mark.parametrize('sets', [1, 2])
def test_nothing_to_do(sets):
    pools, tables = P.make_cache(2, 2, 64, [20, 20], 16, sets)
    lengths = ints(20, 20)
    assert run(queries(2, 0, 4, 64), pools, tables, lengths).shape == (2, 0, 4, 64)
    assert run(queries(0, 1, 4, 64), pools, tables[:0], lengths[:0]).shape == (0, 1, 4, 64)
    assert not run(queries(2, 3, 4, 64), pools, tables[:, :0], lengths).any()


def test_a_second_window_beyond_everything():
    """Windows larger than any sequence: all pairs of keys."""
    lengths = [40, 3]
    pools, tables = P.make_cache(2, 1, 64, lengths, 16, 2)
    for n in (1, 30):
        q = queries(2, n, 2, 64)
        out = run(q, pools, tables, ints(*lengths), w1=1 << 40, w2=1 << 30)
        P.check(out, want(q, pools, tables, lengths, w1=64, w2=64))


def test_replays_of_a_graph():
    """A decode step (rows into pages, both attentions, a token) recorded once and replayed on new inputs, with eager work between the replays."""
    b, h, hk, d, page = 3, 4, 2, 64, 16
    lengths = [40, 700, 1300]
    pools, tables = P.make_cache(b, hk, d, lengths, page, 2)
    at = ints(*lengths)
    q, logits, noise = queries(b, 1, h, d), torch.randn(b, 5000, device='cuda'), torch.rand(b, 5000, device='cuda')
    rows = [torch.randn(b, 1, hk, d, device='cuda', dtype=BF16) for _ in range(4)]

    def step():
        S.paged_append(pools, rows, tables, at)
        dense = S.paged_attn(q, *pools[:2], tables, at)
        pairs = S.paged_two_simplicial_attn(q, pools[:2], pools[2:], tables, at, w1=512, w2=32)
        return dense, pairs, *S.sample_tokens(logits, noise, top_k=50, top_p=0.9)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        recorded = step()
    for replay in range(4):
        q.copy_(queries(b, 1, h, d, seed=replay))
        logits.normal_()
        noise.uniform_()
        for r in rows:
            r.normal_()
        graph.replay()
        got = [t.clone() for t in recorded]
        torch.cuda.synchronize()
        for g, e in zip(got, step()):
            assert torch.equal(g, e)
