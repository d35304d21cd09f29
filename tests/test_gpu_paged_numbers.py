"""2-simplicial attention over paged caches where keys and values are large or no numbers at all: what the definition gives for them."""
import pytest
import torch

import simplicial_attention_amd as S
from tests import paged_util as P

pytestmark = pytest.mark.gpu
BF16, F16 = torch.bfloat16, torch.float16
NAN, INF = float('nan'), float('inf')
# new tokens, heads, second window: one token (few units), units of a wave each, units that share waves
WALKS = [(1, 4, 6), (140, 4, 20), (300, 4, 4)]


def ints(*values):
    return torch.tensor(values, dtype=torch.int32, device='cuda')


def make(n, h, length, d=64, dtype=BF16, seed=11, std=(1., 1., 1., 1.)):
    """Queries, and pools (k1, k2, v1, v2) of one sequence on one key/value head."""
    pools, tables = P.make_cache(1, 1, d, [length], 16, 2, dtype, seed=seed)
    for pool, s in zip(pools, std):
        pool.mul_(s)
    q = torch.randn(1, n, h, d, generator=torch.Generator().manual_seed(seed + 1)).to(dtype).cuda()
    return q, pools, tables


def at(pool, tables, x):
    """The row of position x."""
    return pool[int(tables[0, x // 16]), x % 16, 0]


def compare(q, pools, tables, length, w1, w2, expect=None):
    """NaN, infinities and numbers are where the definition has them, and the numbers agree."""
    got = S.paged_two_simplicial_attn(q, pools[:2], pools[2:], tables, ints(length), w1=w1, w2=w2)
    want = P.attend(q, pools[:2], pools[2:], tables, [length], w1=w1, w2=w2)
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    wide = torch.isinf(want)
    assert torch.equal(torch.isinf(got), wide) and torch.equal(got[wide].double(), want[wide])
    fine = torch.isfinite(want)
    P.check(got[fine], want[fine])
    if expect is not None:
        assert expect(want)


@pytest.mark.parametrize('dtype', [BF16, F16])
@pytest.mark.parametrize('bad', [NAN, INF, -INF])
@pytest.mark.parametrize('n,h,w2', WALKS)
@pytest.mark.parametrize('where', ['q', 'k2', 'one channel of k2'])
def test_what_is_no_number_reaches_the_rows_that_attend_it(where, n, h, w2, bad, dtype):
    length = n + 40
    q, pools, tables = make(n, h, length, dtype=dtype)
    if where == 'q':
        q[0, n // 2, 1, 7] = bad
    else:
        row = at(pools[1], tables, length - 1 - (n - 1) // 2)
        row[7 if where == 'one channel of k2' else slice(None)] = bad
    compare(q, pools, tables, length, 25, w2, lambda want: bool(torch.isnan(want).any()))


@pytest.mark.parametrize('dtype', [BF16, F16])
@pytest.mark.parametrize('n,h,w2', WALKS)
def test_an_infinite_key_that_weighs_nothing(n, h, w2, dtype):
    """Logits of -inf for every pair with one second key: the other pairs share the weight, and every row is a number."""
    length = n + 40
    q, pools, tables = make(n, h, length, dtype=dtype)
    q[..., 7] = 1
    for x in range(length):
        at(pools[0], tables, x)[7] = -1
    at(pools[1], tables, length - 1 - (n - 1) // 2)[7] = INF
    compare(q, pools, tables, length, 25, w2, lambda want: bool(torch.isfinite(want).all()))


@pytest.mark.parametrize('d', [32, 64, 96, 256])
@pytest.mark.parametrize('n,h,w2', WALKS)
def test_products_beyond_the_range_of_fp16(n, h, w2, d):
    """q * k2 of hundreds of thousands against small first keys: ordinary logits, and an ordinary softmax."""
    length = n + 40
    q, pools, tables = make(n, h, length, d, F16, std=(2e-4, 800., 1., 1.))
    q.mul_(800)
    compare(q, pools, tables, length, 25, w2, lambda want: bool(torch.isfinite(want).all()))


@pytest.mark.parametrize('n,h,w2', WALKS)
def test_one_large_channel_keeps_the_digits_of_the_others(n, h, w2):
    """A product of 3.6e9 in a channel that the first keys leave out, beside channels of unit variance; in every fourth second key, so that columns of one wave differ."""
    length = n + 40
    q, pools, tables = make(n, h, length, dtype=F16)
    q[..., 7] = 6e4
    for x in range(length):
        at(pools[0], tables, x)[7] = 0
        at(pools[1], tables, x)[7] = 6e4 if x % 4 == 0 else 1
    compare(q, pools, tables, length, 25, w2, lambda want: bool(torch.isfinite(want).all()))


@pytest.mark.parametrize('scale', [2e-3, 1., 300.])
def test_scales_of_products_beyond_the_range(scale):
    n, length = 30, 60
    q, pools, tables = make(n, 2, length, dtype=F16, std=(2e-4, 300. / scale ** .5, 1., 1.))
    q.mul_(300 / scale ** .5)
    got = S.paged_two_simplicial_attn(q, pools[:2], pools[2:], tables, ints(length), w1=25, w2=6, scale=scale)
    P.check(got, P.attend(q, pools[:2], pools[2:], tables, [length], w1=25, w2=6, scale=scale))
