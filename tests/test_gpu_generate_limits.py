"""Answers from a cache stay inside what the model knows: its positions."""
import pytest
import torch

from simplicial_attention_amd.two_simplicial_transformer import TwoSimplicialLM

pytestmark = pytest.mark.gpu


def model(max_seq_len=64):
    torch.manual_seed(0)
    with torch.device('cuda'):
        lm = TwoSimplicialLM(num_tokens=50, dim=64, depth=2, max_seq_len=max_seq_len, dim_head=32, heads=2, two_simplicial_attn_every=2,
                             transformer_kwargs=dict(key_value_heads=1, two_simplicial_attn_kwargs=dict(w1=16, w2=4)))
    return lm.bfloat16().eval()


def test_tokens_beyond_the_last_position_are_refused():
    lm = model()
    cache = lm.transformer.cache(pages=20, page_size=8)
    long, short = cache.new(), cache.new()
    lm.logits_cached(torch.zeros(2, 60, dtype=torch.long, device='cuda'), cache, cache.extend([long, short], [60, 20]))
    # (the padding of the longer sequence's chunk passes the last position, its tokens do not)
    logits = lm.logits_cached(torch.zeros(2, 9, dtype=torch.long, device='cuda'), cache, cache.extend([long, short], [4, 9]))
    assert bool(torch.isfinite(logits).all())
    with pytest.raises(ValueError, match='64'):
        lm.logits_cached(torch.zeros(2, 1, dtype=torch.long, device='cuda'), cache, cache.extend([long, short], 1))
    with pytest.raises(ValueError):
        lm.generate(torch.zeros(1, 60, dtype=torch.long, device='cuda'), 6)
    tokens, _ = lm.generate(torch.zeros(1, 60, dtype=torch.long, device='cuda'), 5)
    assert tokens.shape == (1, 1, 5)
