"""First windows of any size beside rows in front of a sequence (more rows than tokens)."""
import pytest
import torch

import simplicial_attention_amd as S
from tests import paged_util as P

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('w1', [1 << 40, (1 << 31) - 1, (1 << 31) - 40, 500])
@pytest.mark.parametrize('n,length,w2', [(150, 99, 20), (300, 251, 4), (300, 3, 4), (60, 7, 20)])
def test_rows_in_front_of_a_sequence(n, length, w2, w1):
    """Workgroups that begin in front of the sequence serve their other rows."""
    h = 4
    pools, tables = P.make_cache(1, h, 64, [length], 16, 2, torch.bfloat16, seed=31)
    q = torch.randn(1, n, h, 64, generator=torch.Generator().manual_seed(32)).bfloat16().cuda()
    at = lambda *x: torch.tensor(x, dtype=torch.int32, device='cuda')
    got = S.paged_two_simplicial_attn(q, pools[:2], pools[2:], tables, at(length), at(n), w1=w1, w2=w2)
    P.check(got, P.attend(q, pools[:2], pools[2:], tables, [length], [n], w1=min(w1, 1 << 20), w2=w2))
    assert not got[0, :n - length].any()
