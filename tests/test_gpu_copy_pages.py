"""Page numbers of every integer type are what they say: none wraps around into another page's."""
import pytest
import torch

import simplicial_attention_amd as S
from simplicial_attention_amd import _native

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('pair', [(1 << 32, 1), (0, (1 << 32) + 1), ((1 << 64) - (1 << 32), 2)])
@pytest.mark.parametrize('dtype', [torch.int64, torch.uint64])
def test_numbers_beyond_32_bits_are_refused(pair, dtype):
    if dtype == torch.int64 and max(pair) >= 1 << 63:
        pair = tuple(x - (1 << 64) if x >= 1 << 63 else x for x in pair)
    pool = torch.arange(4 * 6, device='cuda', dtype=torch.float32).view(4, 1, 1, 6)
    before = pool.clone()
    with pytest.raises((ValueError, _native.Sa2Error)):
        S.copy_pages([pool], torch.tensor([pair], dtype=dtype))
    assert torch.equal(pool, before)


@pytest.mark.parametrize('dtype', [torch.uint8, torch.int8, torch.int16, torch.int32, torch.int64, torch.uint16, torch.uint32, torch.uint64])
def test_every_integer_type(dtype):
    pool = torch.arange(4 * 6, device='cuda', dtype=torch.float32).view(4, 1, 1, 6)
    S.copy_pages([pool], torch.tensor([[3, 1]], dtype=dtype))
    assert torch.equal(pool[1], pool[3])


def test_lists_of_numbers_beyond_64_bits_are_refused():
    pool = torch.zeros(4, 1, 1, 6, device='cuda')
    with pytest.raises((ValueError, RuntimeError, OverflowError)):
        S.copy_pages([pool], [(1 << 64, 1)])
