"""The language model's answers from a paged cache against its forward over whole sequences."""
import pytest
import torch

import simplicial_attention_amd as S
from simplicial_attention_amd.two_simplicial_transformer import TwoSimplicialLM

pytestmark = pytest.mark.gpu


def model(dtype=torch.bfloat16, dim_head=64, heads=4, kv_heads=2, w1=24, w2=8, **kw):
    torch.manual_seed(0)
    with torch.device('cuda'):
        lm = TwoSimplicialLM(num_tokens=256, dim=128, depth=4, max_seq_len=256, dim_head=dim_head, heads=heads, two_simplicial_attn_every=2,
                             transformer_kwargs=dict(key_value_heads=kv_heads, two_simplicial_attn_kwargs=dict(w1=w1, w2=w2, **kw)))
    return lm.to(dtype).eval()


# Eight layers round their activations to 8 bits (both sides, at other places): the logits' relative error stays below 2e-2, the bound of the model's training passes
BOUND = 2e-2


def close(a, b):
    assert float((a.double() - b.double()).norm() / b.double().norm()) < BOUND


@pytest.mark.parametrize('kw', [dict(), dict(dim_head=32, heads=8, kv_heads=1), dict(dim_head=40), dict(w2=40), dict(dtype=torch.float32), dict(dtype=torch.float16),
                                dict(dim_head_values=32), dict(qk_rmsnorm=False)], ids=str)
def test_logits_of_chunks_equal_the_whole_forward(kw):
    lm = model(**kw)
    tokens = torch.randint(0, 256, (3, 100), device='cuda')
    lengths = [100, 61, 37]
    whole = [lm(tokens[s:s + 1, :n])[0] for s, n in enumerate(lengths)]
    cache = lm.transformer.cache(pages=20, page_size=16)
    sequences = [cache.new() for _ in lengths]
    got = [[] for _ in lengths]
    at = 0
    for chunk in (33, 1, 1, 40, 25):
        counts = [min(max(n - at, 0), chunk) for n in lengths]
        logits = lm.logits_cached(tokens[:, at:at + chunk], cache, cache.extend(sequences, counts))
        for s, count in enumerate(counts):
            got[s].append(logits[s, :count])
        at += chunk
    for s in range(3):
        close(torch.cat(got[s]), whole[s].detach())


def test_generate_reads_prompts_once_and_forks_them():
    lm = model()
    prompts = torch.randint(0, 256, (2, 50), device='cuda')
    lengths, steps, samples = [50, 23], 40, 3
    make = lambda: torch.Generator(device='cuda').manual_seed(5)
    tokens, logprobs = lm.generate(prompts, steps, lengths=lengths, samples=samples, temperature=0.8, top_k=50, top_p=0.95, min_p=0.01, generator=make(), chunk=20, page_size=16)
    assert tokens.shape == logprobs.shape == (2, samples, steps) and int(tokens.min()) >= 0 and int(tokens.max()) < 256
    again = lm.generate(prompts, steps, lengths=lengths, samples=samples, temperature=0.8, top_k=50, top_p=0.95, min_p=0.01, generator=make(), chunk=20, page_size=16)
    assert torch.equal(again[0], tokens) and torch.equal(again[1], logprobs)
    assert len({tuple(row) for row in tokens.flatten(0, 1).tolist()}) == 2 * samples
    # the log-probabilities are those of the whole forward over prompt and answer
    for s, n in enumerate(lengths):
        for k in range(samples):
            text = torch.cat([prompts[s, :n], tokens[s, k]])[None]
            whole = torch.log_softmax(lm(text)[0, n - 1:-1].float(), -1).gather(1, tokens[s, k][:, None])[:, 0]
            assert float((whole - logprobs[s, k]).abs().max()) < 0.1 and float((whole - logprobs[s, k]).abs().mean()) < 0.02


def test_greedy_answers_do_not_depend_on_pages_and_samples():
    lm = model()
    prompts = torch.randint(0, 256, (1, 30), device='cuda')
    one, _ = lm.generate(prompts, 20, temperature=0., page_size=64)
    three, _ = lm.generate(prompts, 20, samples=3, temperature=0., page_size=8)
    assert torch.equal(three, one.expand(1, 3, 20))


def test_refusals():
    lm = model()
    prompts = torch.randint(0, 256, (2, 30), device='cuda')
    for kw in (dict(steps=0), dict(steps=1, samples=0), dict(steps=1, lengths=[0, 3]), dict(steps=1, lengths=[31, 3]), dict(steps=1, lengths=[3]), dict(steps=300)):
        with pytest.raises(ValueError):
            lm.generate(prompts, **kw)
    cache = lm.transformer.cache(pages=1, page_size=16)
    a = cache.new()
    with pytest.raises(S.OutOfPages):
        cache.extend([a], 17)
