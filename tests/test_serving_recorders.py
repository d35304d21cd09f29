"""The serving functions refuse recorders, which would keep a result's allocation without the kernel that fills it."""
import pytest
import torch
from torch.fx.experimental.proxy_tensor import make_fx

from simplicial_attention_amd import copy_pages, paged_append, paged_attn, paged_two_simplicial_attn, sample_tokens

POOL = torch.zeros(2, 4, 1, 8, dtype=torch.bfloat16)
TABLES, LENGTHS = torch.zeros(1, 2, dtype=torch.int32), torch.ones(1, dtype=torch.int32)


def appended(x):
    paged_append([POOL], [x], TABLES, LENGTHS)
    return x + 1


def copied(x):
    copy_pages([POOL], [(0, 1)])
    return x + 1


CALLS = {
    'paged_attn': lambda x: paged_attn(x, POOL, POOL, TABLES, LENGTHS),
    'paged_two_simplicial_attn': lambda x: paged_two_simplicial_attn(x, (POOL, POOL), (POOL, POOL), TABLES, LENGTHS),
    'paged_append': appended,
    'copy_pages': copied,
    'sample_tokens': lambda x: sample_tokens(x.float(), torch.ones(x.shape))[1],
}


# (on host tensors, which each call refuses too: the recorder has to be noticed first)
@pytest.mark.parametrize('name', CALLS)
@pytest.mark.parametrize('record', [lambda f, x: torch.jit.trace(f, x, check_trace=False), lambda f, x: make_fx(f)(x)], ids=['trace', 'make_fx'])
def test_recorders_are_refused(name, record):
    with torch.no_grad(), pytest.raises(RuntimeError, match='cannot be traced'):
        record(CALLS[name], torch.zeros(1, 1, 1, 8, dtype=torch.bfloat16))
