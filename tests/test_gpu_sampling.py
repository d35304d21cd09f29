"""Next tokens from logits and given random numbers."""
import math

import pytest
import torch

import simplicial_attention_amd as S
from tests import paged_util as P

pytestmark = pytest.mark.gpu
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
INF = math.inf


def check(logits, noise, temperature=1., top_k=0, top_p=1., min_p=0.):
    """Tokens equal the definition's in 64 bits (random draws come within 1e-5 of a tie or a threshold once in 10^4 rows: the seeds here do not), log-probabilities agree
    to fp32 sums: the terms' errors of 2^-22 relative and the logarithm's."""
    rows = len(logits)
    column = lambda v: [float(x) for x in v] if torch.is_tensor(v) else [v] * rows
    tokens, logprobs = S.sample_tokens(logits, noise, temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p)
    want, want_lp = P.sample(logits.cpu(), noise.cpu(), column(temperature), column(top_k), column(top_p), column(min_p))
    assert tokens.dtype == torch.int64 and logprobs.dtype == torch.float32
    assert torch.equal(tokens.cpu(), want)
    fine = torch.isfinite(want_lp)
    assert torch.equal(torch.isfinite(logprobs.cpu()), fine)
    assert bool(((logprobs.cpu().double() - want_lp)[fine].abs() <= 2e-6 * (1 + want_lp[fine].abs()) + 2. ** -22 * logits.float().cpu().nan_to_num(0, 0, 0).abs().amax()).all())
    return tokens


def inputs(rows, vocab, dtype, seed=0, std=2.5):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(rows, vocab, generator=g) * std).to(dtype).cuda(), torch.rand(rows, vocab, generator=g).cuda()


@pytest.mark.parametrize('dtype', [F32, BF16, F16])
@pytest.mark.parametrize('rows, vocab', [(1, 1), (3, 2), (8, 256), (5, 63), (4, 1000), (2, 2049), (3, 50257), (2, 131072), (40, 300)])
def test_without_filters(rows, vocab, dtype):
    logits, noise = inputs(rows, vocab, dtype)
    check(logits, noise)
    check(logits, noise, temperature=0.7)
    assert torch.equal(check(logits, noise, temperature=0.).cpu(), logits.float().cpu().sort(dim=-1, descending=True, stable=True).indices[:, 0])


@pytest.mark.parametrize('dtype', [F32, BF16])
@pytest.mark.parametrize('filters', [dict(top_k=1), dict(top_k=5), dict(top_k=10 ** 6), dict(top_p=0.), dict(top_p=0.3), dict(top_p=0.95), dict(top_p=7.), dict(min_p=0.05),
                                     dict(min_p=1.), dict(top_k=40, top_p=0.8, min_p=0.02)], ids=str)
@pytest.mark.parametrize('rows, vocab', [(16, 256), (6, 5000), (3, 100001)])
def test_filters(rows, vocab, filters, dtype):
    for seed, std in ((1, 2.5), (2, 0.1)):
        logits, noise = inputs(rows, vocab, dtype, seed, std)
        check(logits, noise, temperature=1.3, **filters)


@pytest.mark.parametrize('vocab', [256, 40000])
def test_parameters_of_each_row(vocab):
    rows = 24
    logits, noise = inputs(rows, vocab, BF16, 3)
    g = torch.Generator().manual_seed(4)
    rand = lambda: torch.rand(rows, generator=g).cuda()
    check(logits, noise, temperature=rand() * 2 * (rand() > 0.2), top_k=(rand() * 60).int(), top_p=rand() * 1.2, min_p=0.2 * rand())


def test_ties_keep_the_lowest_index():
    """Equal logits are ordered by index: top-k, top-p and the greedy choice all cut inside a tie."""
    noise = torch.rand(64, 1000, generator=torch.Generator().manual_seed(5)).cuda()
    logits = torch.zeros(64, 1000, device='cuda')
    for kw in (dict(top_k=3), dict(top_p=0.0045), dict(top_k=700, top_p=0.5)):
        most = {3: 3, 700: 500}.get(kw.get('top_k'), 5)
        tokens, _ = S.sample_tokens(logits, noise, **kw)
        assert int(tokens.max()) < most
        want = (-torch.log(-torch.log(noise[:, :most].double()))).argmax(-1)
        assert torch.equal(tokens, want)
    assert not S.sample_tokens(logits, noise, temperature=0.)[0].any()
    logits[:, 10:] = 1
    assert bool((S.sample_tokens(logits, noise, temperature=0.)[0] == 10).all())


def test_logits_at_the_edges():
    """Masked vocabularies, rows without any token, infinities and NaN, random numbers of 0 and 1."""
    logits, noise = inputs(8, 500, F32, 6)
    logits[0] = -INF
    logits[1] = float('nan')
    logits[2, 7:] = -INF
    logits[3, ::2] = float('nan')
    logits[4, 33] = INF
    logits[5] = -3e38
    logits[6, 100:] = torch.finfo(F32).min
    noise[7, :250], noise[7, 250:] = 0, 1
    tokens = check(logits, noise)
    assert tokens[0] == -1 and tokens[1] == -1 and 0 <= tokens[2] < 7 and tokens[3] % 2 == 1 and tokens[4] == 33 and 0 <= tokens[6] < 100
    check(logits, noise, temperature=1e-30)
    check(logits, noise, temperature=0.)
    check(logits, noise, top_k=4, top_p=0.5, min_p=0.1)


def test_strides_shapes_and_streams():
    logits, noise = inputs(6, 2 * 777, BF16, 7)
    check(logits[:, 1:778], noise[:, 5:782])
    check(logits[::2, ::2], noise[::2, ::2])
    shaped, lp = S.sample_tokens(logits.view(2, 3, -1), noise.view(2, 3, -1), temperature=0.9)
    flat, lp2 = S.sample_tokens(logits, noise, temperature=0.9)
    assert shaped.shape == (2, 3) and torch.equal(shaped.flatten(), flat) and torch.equal(lp.flatten(), lp2)
    one, _ = S.sample_tokens(logits[0], noise[0], temperature=0.9)
    assert one.shape == () and one == flat[0]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        other, _ = S.sample_tokens(logits, noise, temperature=0.9)
    torch.cuda.current_stream().wait_stream(stream)
    assert torch.equal(other, flat)
    assert S.sample_tokens(logits[:0], noise[:0])[0].shape == (0,)


def test_draws_follow_the_distribution():
    """Frequencies of 20000 draws from 8 tokens against the kept probabilities: within 4.5 standard deviations (one in 10^5 each)."""
    n = 20000
    x = torch.tensor([2., 1., 0.5, 0., -1., -1.5, -3., 1.5], device='cuda')
    noise = torch.rand(n, 8, generator=torch.Generator().manual_seed(8)).cuda()
    for kw, kept in ((dict(), 8), (dict(top_k=4), 4), (dict(top_p=0.6), 2)):
        tokens, _ = S.sample_tokens(x.expand(n, 8), noise, **kw)
        order = x.argsort(descending=True)[:kept]
        p = torch.zeros(8, dtype=torch.float64, device='cuda')
        p[order] = torch.softmax(x[order].double(), -1)
        f = torch.bincount(tokens, minlength=8).double() / n
        assert bool(((f - p).abs() <= 4.5 * (p * (1 - p) / n).sqrt()).all()), (f, p)


def test_refusals():
    logits, noise = inputs(4, 100, F32)
    with pytest.raises(AssertionError):
        S.sample_tokens(logits.cpu(), noise.cpu())
    with pytest.raises(TypeError):
        S.sample_tokens(logits.double(), noise)
    with pytest.raises(TypeError):
        S.sample_tokens(logits, noise.half())
    with pytest.raises(ValueError):
        S.sample_tokens(logits, noise[:, :99])
    with pytest.raises(ValueError):
        S.sample_tokens(logits[:, :0], noise[:, :0])
    with pytest.raises(ValueError):
        S.sample_tokens(logits, noise, temperature=-1.)
    with pytest.raises(ValueError):
        S.sample_tokens(logits, noise, top_p=math.nan)
    with pytest.raises(TypeError):
        S.sample_tokens(logits, noise, top_k=torch.ones(4, device='cuda'))
    with pytest.raises(ValueError):
        S.sample_tokens(logits, noise, temperature=torch.ones(3, device='cuda'))
    with pytest.raises(RuntimeError):
        S.sample_tokens(logits.requires_grad_(), noise)
