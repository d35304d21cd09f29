"""Sizes whose product passes 64 bits are refused like other sizes beyond a launch: no product wraps around into a small one."""
import os

import pytest

from simplicial_attention_amd import _native
from tests.test_serving_abi import index, pool, problem, rows


@pytest.fixture(scope='module')
def lib():
    if not os.path.exists(_native.LIB_PATH):
        _native.build()
    return _native.load()


SIZES = [(1 << 22, 1 << 21, 1 << 21), (1 << 30, 1 << 30, 1 << 4), (1 << 30, 1 << 30, 1 << 30), ((1 << 31) - 1, (1 << 31) - 1, (1 << 31) - 1), (1 << 26, 1, 1)]


@pytest.mark.parametrize('batch,n,heads', SIZES)
def test_attention_refuses(lib, batch, n, heads):
    prob, t, p = problem(batch=batch, rows=n, heads=heads, kv_heads=1), rows(), pool()
    assert lib.sa2_paged_attn_workspace_bytes(prob) == -1 and lib.sa2_paged_simplicial_attn_workspace_bytes(prob) == -1
    assert lib.sa2_paged_attn(prob, t, p, p, index(), t, None, 0, None) == 2
    assert 'too large' in lib.sa2_last_error().decode()
    assert lib.sa2_paged_simplicial_attn(prob, t, p, p, p, p, index(), t, None, 0, None) == 2


@pytest.mark.parametrize('batch,n,heads', SIZES[:-1])
def test_append_refuses(lib, batch, n, heads):
    prob = problem(batch=batch, rows=n, heads=heads, kv_heads=heads)
    assert lib.sa2_paged_append(prob, (_native.AppendItem * 1)(_native.AppendItem(pool(), rows())), 1, 0, index(), None) == 2
    assert 'too large' in lib.sa2_last_error().decode()


def test_sampling_refuses(lib):
    for n in (1 << 31, 1 << 50, (1 << 63) - 1):
        assert lib.sa2_sample_workspace_bytes(n, 1 << 24) == -1 and lib.sa2_sample_workspace_bytes(n, 100) == -1
    assert lib.sa2_sample_workspace_bytes((1 << 31) - 1, 100) == 0
