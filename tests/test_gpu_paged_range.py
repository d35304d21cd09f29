"""Attention over paged caches where every logit is far from zero: a softmax is one whatever its logits' size."""
import pytest
import torch

import simplicial_attention_amd as S
from tests import paged_util as P

pytestmark = pytest.mark.gpu


def ints(*values):
    return torch.tensor(values, dtype=torch.int32, device='cuda')


@pytest.mark.parametrize('dtype,size', [(torch.bfloat16, 1e14), (torch.bfloat16, 1e16), (torch.bfloat16, 1e18), (torch.float16, 6e4)])
@pytest.mark.parametrize('sign', [-1, 1])
@pytest.mark.parametrize('n,h,length', [(1, 4, 1), (1, 4, 300), (20, 4, 60), (20, 1, 20), (300, 4, 340)])
@pytest.mark.parametrize('sets', [1, 2])
def test_logits_far_from_zero(sets, n, h, length, sign, dtype, size):
    """Logits of size^2 / 8 and half of that, of one sign: the keys of the larger ones share the weight."""
    pools, tables = P.make_cache(1, 1, 64, [length], 16, sets, dtype, seed=51)
    x = torch.arange(length, device='cuda')
    k1 = pools[0][tables[0].long()[x // 16], x % 16]
    k1.zero_()
    k1[:, 0, 9] = (sign * torch.where(x % 3 == 0, size / 2, size)).to(dtype)
    pools[0][tables[0].long()[x // 16], x % 16] = k1
    if sets == 2:
        pools[1][tables[0].long()[x // 16], x % 16, 0, 9] = 1
    q = torch.randn(1, n, h, 64, generator=torch.Generator().manual_seed(52)).to(dtype).cuda()
    q[..., 9] = size
    for w2 in (4, 20) if sets == 2 else (None,):
        kw = {} if sets == 1 else dict(w1=30, w2=w2)
        if sets == 1:
            got = S.paged_attn(q, *pools, tables, ints(length))
        else:
            got = S.paged_two_simplicial_attn(q, pools[:2], pools[2:], tables, ints(length), **kw)
        P.check(got, P.attend(q, pools[:sets], pools[sets:], tables, [length], **kw))
