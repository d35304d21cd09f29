"""The type of a cache is the caller's choice where the weights have none that pools can hold."""
import pytest
import torch

from simplicial_attention_amd import PagedCache
from simplicial_attention_amd.two_simplicial_transformer import TwoSimplicialLM, TwoSimplicialTransformer

pytestmark = pytest.mark.gpu


def model(dtype):
    torch.manual_seed(0)
    with torch.device('cuda'):
        lm = TwoSimplicialLM(num_tokens=50, dim=64, depth=4, max_seq_len=128, dim_head=32, heads=2, two_simplicial_attn_every=4,
                             transformer_kwargs=dict(key_value_heads=1, two_simplicial_attn_kwargs=dict(w1=16, w2=4)))
    return lm.to(dtype).eval()


@pytest.mark.parametrize('weights,cache,expected', [(torch.float32, None, torch.bfloat16), (torch.float32, torch.float16, torch.float16), (torch.float32, torch.bfloat16, torch.bfloat16),
                                                    (torch.bfloat16, None, torch.bfloat16), (torch.float16, None, torch.float16), (torch.bfloat16, torch.float16, torch.float16)])
def test_generate_takes_the_caches_type(monkeypatch, weights, cache, expected):
    lm, made = model(weights), []
    original = TwoSimplicialTransformer.cache
    monkeypatch.setattr(TwoSimplicialTransformer, 'cache', lambda self, *a, **kw: made.append(original(self, *a, **kw)) or made[-1])
    tokens, logprobs = lm.generate(torch.zeros(2, 20, dtype=torch.long, device='cuda'), 6, temperature=0., **({} if cache is None else {'dtype': cache}))
    assert tokens.shape == (2, 1, 6) and bool(torch.isfinite(logprobs).all())
    assert len(made) == 1 and {pool.dtype for pool in made[0].pools} == {expected}
    with pytest.raises(TypeError):
        lm.generate(torch.zeros(2, 20, dtype=torch.long, device='cuda'), 6, dtype=torch.float32)


# Roundings of a dense layer in fp32 whose rows are in a cache: q, k, v, the weights and the output, each of a relative error of at most half an ulp (2^-9 in bf16, 2^-12 in fp16; rms
# 0.6 of that).  Those of q and k enter through logits below 1, the five are independent: below 3 * 2^-9 (2^-12) of the result's norm.
@pytest.mark.parametrize('dtype,bound', [(torch.bfloat16, 3 * 2. ** -9), (torch.float16, 3 * 2. ** -12)])
def test_a_dense_layer_in_fp32_is_rounded_to_its_cache(dtype, bound):
    layer = model(torch.float32).transformer.layers[0][0]
    x = torch.randn(2, 50, 64, generator=torch.Generator().manual_seed(1)).cuda()
    cache = PagedCache([(1, 1, 32)], pages=20, page_size=8, dtype=dtype)
    batch = cache.extend([cache.new(), cache.new()], 50)
    with torch.no_grad():
        whole = layer(x)
    got = layer.forward_cached(x, cache.keys[0], cache.values[0], batch)
    assert got.dtype == torch.float32
    assert float((got - whole).norm() / whole.norm()) < bound
