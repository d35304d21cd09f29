"""Sampling parameters per row that are infinite or no numbers (numbers for all rows are checked on the host)."""
import math

import pytest
import torch

import simplicial_attention_amd as S
from tests import paged_util as P

pytestmark = pytest.mark.gpu
INF, NAN = math.inf, math.nan


def inputs(vocab, seed, masked):
    g = torch.Generator().manual_seed(seed)
    logits, noise = torch.randn(12, vocab, generator=g) * 2, torch.rand(12, vocab, generator=g)
    if masked:
        logits[:, 1::2] = -INF
    return logits.cuda(), noise.cuda()


def rows_of(value, dtype=torch.float32):
    return torch.full((12,), value, dtype=dtype, device='cuda')


@pytest.mark.parametrize('vocab', [300, 3000, 20000])
@pytest.mark.parametrize('masked', [False, True])
@pytest.mark.parametrize('filters', [dict(), dict(top_p=0.5), dict(top_k=30), dict(top_k=30, top_p=0.7, min_p=0.5)], ids=str)
def test_an_infinite_temperature_draws_evenly(vocab, masked, filters):
    """All tokens that are there weigh the same: what a temperature of 1e30 gives in 64 bits."""
    logits, noise = inputs(vocab, 41, masked)
    per_row = {k: rows_of(v, torch.int32 if k == 'top_k' else torch.float32) for k, v in filters.items()}
    tokens, logprobs = S.sample_tokens(logits, noise, temperature=rows_of(INF), **per_row)
    column = lambda k, default: [float(per_row[k][0]) if k in per_row else default] * 12
    want, want_lp = P.sample(logits.cpu(), noise.cpu(), [1e30] * 12, column('top_k', 0), column('top_p', 1.), column('min_p', 0.))
    assert torch.equal(tokens.cpu(), want)
    assert float((logprobs.cpu().double() - want_lp).abs().max()) < 1e-4


@pytest.mark.parametrize('vocab', [300, 3000, 20000])
@pytest.mark.parametrize('name', ['temperature', 'top_p', 'min_p'])
@pytest.mark.parametrize('other', [dict(), dict(top_k=rows_of)], ids=['alone', 'with top_k'])
def test_a_parameter_that_is_no_number_keeps_the_first_token(vocab, name, other):
    logits, noise = inputs(vocab, 42, True)
    tokens, _ = S.sample_tokens(logits, noise, **{name: rows_of(NAN)}, **({'top_k': rows_of(7, torch.int32)} if other else {}))
    assert torch.equal(tokens, logits.argmax(-1))
