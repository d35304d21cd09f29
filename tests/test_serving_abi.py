"""The serving functions of the C ABI refuse, before any launch, what their kernels do not cover, and say how much workspace they want."""
import ctypes
import os

import pytest

from simplicial_attention_amd import _native


@pytest.fixture(scope='module')
def lib():
    if not os.path.exists(_native.LIB_PATH):
        _native.build()
    return _native.load()


def problem(**changes):
    fields = dict(batch=2, rows=3, heads=4, kv_heads=2, dim_head=64, pool_dim=64, page_size=16, pages=8, table_width=4, w1=32, w2=8, max_length=0, scale=.125, dtype=0)
    fields.update(changes)
    return _native.PagedProblem(**fields)


def rows(ptr=0x1000, sb=768, sn=256, sh=64):
    return _native.TensorArg(ptr, sb, sn, sh)


def pool(ptr=0x2000, page=2048, row=128, head=64):
    return _native.Pool(ptr, page, row, head)


def index(tables=0x3000, lengths=0x4000, counts=None):
    return _native.PagedIndex(tables, 4, lengths, counts)


def text(lib):
    return lib.sa2_last_error().decode()


BAD = [('batch', 0, 2), ('rows', 0, 2), ('heads', 3, 2), ('kv_heads', 0, 2), ('dim_head', 60, 3), ('dim_head', 72, 3), ('pool_dim', 264, 3), ('page_size', 0, 2),
       ('pages', 0, 2), ('table_width', 0, 2), ('max_length', -1, 2), ('scale', 0., 2), ('scale', float('nan'), 2), ('dtype', 2, 3), ('rows', 1 << 28, 2)]


@pytest.mark.parametrize('field,value,code', BAD)
def test_attention_refuses_shapes(lib, field, value, code):
    prob, t, p, at = problem(**{field: value}), rows(), pool(), index()
    assert lib.sa2_paged_attn(prob, t, p, p, at, t, None, 0, None) == code
    assert text(lib) != ''
    assert lib.sa2_paged_attn_workspace_bytes(prob) == -1
    assert lib.sa2_paged_simplicial_attn(prob, t, p, p, p, p, at, t, None, 0, None) == code
    assert lib.sa2_paged_simplicial_attn_workspace_bytes(prob) == -1


def test_attention_refuses_pointers_strides_and_windows(lib):
    prob, t, p, at = problem(), rows(), pool(), index()
    dense = lambda q=t, k=p, v=p, at=at, out=t, prob=prob: lib.sa2_paged_attn(prob, q, k, v, at, out, None, 0, None)
    assert dense(prob=None) == 1 and dense(q=None) == 1 and dense(k=None) == 1 and dense(v=None) == 1 and dense(at=None) == 1 and dense(out=None) == 1
    assert dense(at=index(tables=None)) == 1 and dense(at=index(lengths=None)) == 1
    assert dense(q=rows(ptr=0x1008)) == 4 and dense(out=rows(sn=260)) == 4 and dense(k=pool(ptr=0x2004)) == 4 and dense(v=pool(row=132)) == 4
    assert 'v' in text(lib)
    simp = lambda prob=prob, k2=p, v2=p: lib.sa2_paged_simplicial_attn(prob, t, p, k2, p, v2, at, t, None, 0, None)
    assert simp(k2=None) == 1 and simp(v2=None) == 1 and simp(v2=pool(head=4)) == 4
    assert simp(prob=problem(w1=0)) == 2 and simp(prob=problem(w2=0)) == 2
    assert 'w2' in text(lib)


def test_attention_wants_its_workspace(lib):
    t, p, at = rows(), pool(), index()
    small = problem()
    assert lib.sa2_paged_attn_workspace_bytes(small) == 0 and lib.sa2_paged_simplicial_attn_workspace_bytes(small) == 0
    # one token over a long cache is shared out; so are second windows of more than one block of 32 offsets (three of them: 70)
    long = problem(batch=1, rows=1, pages=4096, table_width=4096)
    need = lib.sa2_paged_attn_workspace_bytes(long)
    assert need > 0 and need % (4 * (64 * 4 + 8)) == 0
    assert lib.sa2_paged_attn(long, t, p, p, at, t, None, 0, None) == 2
    assert str(need) in text(lib)
    assert lib.sa2_paged_attn(long, t, p, p, at, t, 0x8000, need - 1, None) == 2
    assert lib.sa2_paged_attn(long, t, p, p, at, t, 0x8008, need, None) == 4
    # a known length makes it less, and never more
    assert lib.sa2_paged_attn_workspace_bytes(problem(batch=1, rows=1, pages=4096, table_width=4096, max_length=100)) == 0
    wide = problem(batch=1, rows=1, pages=64, table_width=64, w1=32, w2=70)
    assert lib.sa2_paged_simplicial_attn_workspace_bytes(wide) == 3 * 4 * (64 * 4 + 8)
    # ... of which the tables name 64 positions
    assert lib.sa2_paged_simplicial_attn_workspace_bytes(problem(batch=1, rows=1, w2=1 << 30)) == 2 * 4 * (64 * 4 + 8)


def test_append_refuses(lib):
    def call(prob=None, items=None, count=1, src=0, at=None):
        items = [_native.AppendItem(pool(), rows())] if items is None else items
        array = (_native.AppendItem * max(len(items), 1))(*items)
        return lib.sa2_paged_append(problem() if prob is None else prob, array, count, src, index() if at is None else at, None)

    assert call(at=index(tables=None)) == 1 and call(at=index(lengths=None)) == 1
    assert lib.sa2_paged_append(None, (_native.AppendItem * 1)(), 1, 0, index(), None) == 1
    assert call(items=[_native.AppendItem(pool(ptr=None), rows())]) == 1 and call(items=[_native.AppendItem(pool(), rows(ptr=None))]) == 1
    assert call(count=0) == 2 and call(count=5) == 2
    assert call(src=3) == 3 and call(prob=problem(dtype=2)) == 3
    assert call(items=[_native.AppendItem(pool(row=4), rows())]) == 4
    for field, value in (('batch', 0), ('rows', 0), ('kv_heads', 0), ('page_size', 0), ('pages', 0), ('table_width', 0), ('dim_head', 65), ('pool_dim', 260)):
        assert call(prob=problem(**{field: value})) == 2, field


def test_copy_refuses(lib):
    def call(pairs, ptr=0x1000, stride=4096, size=4096, pages=8, n=None):
        flat = [x for pair in pairs for x in pair]
        host = (ctypes.c_int32 * max(len(flat), 1))(*flat)
        return lib.sa2_copy_pages((_native.PagePool * 1)(_native.PagePool(ptr, stride, size, pages)), 1, host, len(pairs) if n is None else n, None)

    assert call([(0, 1)], ptr=None) == 1
    assert lib.sa2_copy_pages(None, 1, None, 0, None) == 1
    assert call([(0, 1)], size=3) == 2 and call([(0, 1)], stride=4094) == 2 and call([(0, 1)], pages=0) == 2
    for pairs in ([(0, 8)], [(-1, 1)], [(0, 1), (2, 1)], [(0, 1), (1, 2)], [(3, 3)], [(1, 2), (0, 1)]):
        assert call(pairs) == 2, pairs
    # more pairs than a page can be written once for, whatever the list says
    assert call([(0, 1)], n=1 << 62) == 2
    assert call([], n=-1) == 2 and call([]) == 0


def test_sample_refuses(lib):
    params = _native.SampleParams(None, None, None, None, 1., 1., 0., 0)

    def call(logits=0x1000, kind=0, n=4, vocab=100, noise=0x2000, params=params, tokens=0x3000, logprobs=0x4000, workspace=None, size=0):
        return lib.sa2_sample(logits, kind, n, vocab, vocab, noise, vocab, params, tokens, logprobs, workspace, size, None)

    assert call(logits=None) == 1 and call(noise=None) == 1 and call(params=None) == 1 and call(tokens=None) == 1 and call(logprobs=None) == 1
    assert call(n=0) == 2 and call(vocab=0) == 2 and call(vocab=(1 << 24) + 1) == 2 and call(n=1 << 30) == 2
    assert call(kind=3) == 3
    assert call(logits=0x1001) == 4 and call(logits=0x1002, kind=2) == 4 and call(noise=0x2002) == 4
    assert lib.sa2_sample_workspace_bytes(4, 4096) == 0 and lib.sa2_sample_workspace_bytes(0, 10) == -1
    need = lib.sa2_sample_workspace_bytes(4, 4097)
    assert need > 0
    assert call(vocab=4097) == 2 and call(vocab=4097, workspace=0x5000, size=need - 1) == 2 and call(vocab=4097, workspace=0x5008, size=need) == 4
