"""2-simplicial attention over paged caches: values that are no numbers, beside columns that hold nothing that counts."""
import pytest
import torch

import simplicial_attention_amd as S
from tests import paged_util as P

pytestmark = pytest.mark.gpu
NAN, INF = float('nan'), float('inf')
# new tokens, heads, second windows: one token (few units), units of a wave each, units that share waves
WALKS = [(1, 4, 6), (1, 4, 1), (140, 4, 20), (140, 4, 1), (300, 4, 4), (300, 4, 1)]


def ints(*values):
    return torch.tensor(values, dtype=torch.int32, device='cuda')


def make(n, h, length, dtype, positive=()):
    pools, tables = P.make_cache(1, 1, 64, [length], 16, 2, dtype, seed=21)
    for i in positive:
        pools[i].abs_()
    return torch.randn(1, n, h, 64, generator=torch.Generator().manual_seed(22)).to(dtype).cuda(), pools, tables


def at(pool, tables, x):
    return pool[int(tables[0, x // 16]), x % 16, 0]


def compare(q, pools, tables, length, w1, w2):
    got = S.paged_two_simplicial_attn(q, pools[:2], pools[2:], tables, ints(length), w1=w1, w2=w2)
    want = P.attend(q, pools[:2], pools[2:], tables, [length], w1=w1, w2=w2)
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    wide = torch.isinf(want)
    assert torch.equal(torch.isinf(got), wide) and torch.equal(got[wide].double(), want[wide])
    fine = torch.isfinite(want)
    P.check(got[fine], want[fine])
    return want


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float16])
@pytest.mark.parametrize('which', ['v1', 'v2'])
@pytest.mark.parametrize('n,h,w2', WALKS)
def test_infinite_values_stay_infinite(n, h, w2, which, dtype):
    """One infinite value among positive ones: the rows that attend it are infinite in its channel."""
    length = n + 40
    q, pools, tables = make(n, h, length, dtype, positive=(2, 3))
    at(pools[2 if which == 'v1' else 3], tables, length - 1 - (n - 1) // 2)[5] = INF
    want = compare(q, pools, tables, length, 40, w2)
    assert bool(torch.isinf(want).any()) and not bool(torch.isnan(want).any())


@pytest.mark.parametrize('bad', [NAN, INF])
@pytest.mark.parametrize('n,w2', [(1, 20), (140, 20), (300, 16)])
def test_rows_without_first_keys_are_zero(n, w2, bad):
    """The page of a first window is missing, and the longer second window holds a value that is no number."""
    h, length = 4, 160 if n == 1 else n
    q, pools, tables = make(n, h, length, torch.bfloat16, positive=(2,))
    page = (length - 1) // 16 if n == 1 else 4
    at(pools[3], tables, 16 * page - 4)[:] = bad
    tables[0, page] = -1
    want = compare(q, pools, tables, length, 4, w2)
    rows = slice(None) if n == 1 else slice(16 * page + 3, 16 * page + 16)
    assert not bool(want[0, rows].any())
