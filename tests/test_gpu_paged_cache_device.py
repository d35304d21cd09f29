"""A cache's tables go where its pools are, whichever device is current when they are made."""
import pytest
import torch

import simplicial_attention_amd as S

pytestmark = pytest.mark.gpu


def test_a_cache_knows_the_device_of_its_pools():
    for device in ('cuda', 'cuda:0', torch.device('cuda')):
        cache = S.PagedCache([(1, 1, 8), (2, 2, 16)], pages=4, page_size=4, device=device)
        assert all(cache.device == pool.device for pool in cache.pools)
        batch = cache.extend([cache.new()], 3)
        assert batch.tables.device == batch.lengths.device == batch.counts.device == cache.pools[0].device
