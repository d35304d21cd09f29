"""Which page belongs to whom: the host side of the paged cache, on the CPU.  The page copies are recorded and played on the CPU pools."""
import random

import pytest
import torch

import simplicial_attention_amd as S
from simplicial_attention_amd import paged


@pytest.fixture
def cache(monkeypatch):
    def play(pools, pairs):
        written = [dst for _, dst in pairs]
        assert len(set(written)) == len(written) and not set(written) & {src for src, _ in pairs}
        for pool in pools:
            for src, dst in pairs:
                pool[dst] = pool[src]
    monkeypatch.setattr(paged, 'copy_pages', play)
    monkeypatch.setattr(torch.Tensor, 'pin_memory', lambda t: t)
    return lambda pages, page_size=4, layers=((1, 1, 8), (2, 2, 16)): S.PagedCache(layers, pages=pages, page_size=page_size, device='cpu')


def write(cache, sequences, counts, marks):
    """Extends and writes the mark of every new token into all pools, as paged_append would."""
    batch = cache.extend(sequences, counts)
    for s, (sequence, count) in enumerate(zip(sequences, counts)):
        length = int(batch.lengths[s])
        assert length == cache.length(sequence) and int(batch.counts[s]) == count and batch.max_length >= length
        for t in range(count):
            x = length - count + t
            page = int(batch.tables[s, x // cache.page_size])
            for pool in cache.pools:
                pool[page, x % cache.page_size] = marks[sequence][x]


def read(cache, sequence):
    table = cache.table(sequence)
    got = [[float(pool[table[x // cache.page_size], x % cache.page_size].flatten()[0]) for x in range(cache.length(sequence))] for pool in cache.pools]
    assert all(g == got[0] for g in got)
    return got[0]


def test_random_lives_of_sequences(cache):
    rng = random.Random(3)
    c = cache(40)
    marks = {}
    serial = 0
    for step in range(600):
        what = rng.choice(['new', 'extend', 'extend', 'extend', 'fork', 'fork', 'free', 'truncate', 'compact'])
        names = list(marks)
        if what == 'new' and len(names) < 8:
            marks[c.new()] = []
        elif what == 'extend' and names:
            some = rng.sample(names, rng.randint(1, len(names)))
            counts = [rng.choice([0, 1, 1, 3, 9]) for _ in some]
            before = {s: (list(c.table(s)), c.length(s)) for s in names}
            trial = {s: marks[s] + [float((serial + 10 * i + t) % 251) for t in range(n)] for i, (s, n) in enumerate(zip(some, counts))}
            serial += 97
            try:
                write(c, some, counts, trial)
                marks.update(trial)
            except S.OutOfPages:
                assert {s: (c.table(s), c.length(s)) for s in names} == before
        elif what == 'fork' and names and len(names) < 12:
            s = rng.choice(names)
            marks[c.fork(s)] = list(marks[s])
        elif what == 'free' and names:
            some = rng.sample(names, rng.randint(1, min(3, len(names))))
            c.free(*some)
            for s in some:
                del marks[s]
        elif what == 'truncate' and names:
            s = rng.choice(names)
            n = rng.randint(0, len(marks[s]))
            c.truncate(s, n)
            del marks[s][n:]
        elif what == 'compact':
            c.compact()
            used = c.pages - c.free_pages
            assert all(page < used for s in marks for page in c.table(s))
        for s in marks:
            assert read(c, s) == marks[s]
        held = {page for s in marks for page in c.table(s)}
        assert c.free_pages == c.pages - len(held)


def test_a_shared_page_is_copied_once_per_writer_but_the_last(cache):
    c = cache(10)
    marks = {}
    a = c.new()
    marks[a] = [1., 2., 3., 4., 5.]
    write(c, [a], [5], marks)
    forks = [c.fork(a) for _ in range(2)]
    assert c.free_pages == 8                              # nothing is copied by a fork
    for i, f in enumerate(forks):
        marks[f] = marks[a] + [10. + i]
    marks[a] = marks[a] + [6.]
    write(c, [a, *forks], [1, 1, 1], marks)
    assert c.free_pages == 6                              # two copies of the partly filled page; the full one is shared still
    assert len({c.table(s)[0] for s in (a, *forks)}) == 1 and len({c.table(s)[1] for s in (a, *forks)}) == 3
    for s in (a, *forks):
        assert read(c, s) == marks[s]


def test_running_out_changes_nothing(cache):
    c = cache(3)
    a, b = c.new(), c.new()
    c.extend([a], [8])
    f = c.fork(a)
    c.extend([b], [1])
    with pytest.raises(S.OutOfPages):
        c.extend([a, f], [1, 0])
    assert c.length(a) == 8 and c.length(f) == 8 and c.free_pages == 0 and c.table(a) == c.table(f)
    c.free(b)
    c.extend([a], [1])


def test_refusals(cache):
    c = cache(4)
    a = c.new()
    c.extend([a], 3)
    for call in (lambda: c.free(99), lambda: c.fork(99), lambda: c.extend([99], [1]), lambda: c.length(99)):
        with pytest.raises(KeyError):
            call()
    for call in (lambda: c.free(a, a), lambda: c.extend([a, a], [1, 1]), lambda: c.extend([a], [-1]), lambda: c.extend([a], [1, 2]), lambda: c.truncate(a, 4),
                 lambda: c.truncate(a, -1), lambda: S.PagedCache([(1, 1, 8)], pages=0, device='cpu')):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(TypeError):
        S.PagedCache([(1, 1, 8)], pages=2, dtype=torch.float32, device='cpu')
    assert c.length(a) == 3
    c.free(a)
    assert c.free_pages == 4
    with pytest.raises(KeyError):
        c.length(a)


def test_channels_are_whole_pieces(cache):
    c = cache(2, layers=((1, 3, 37), (2, 1, 64)))
    assert [tuple(p.shape) for p in c.pools] == [(2, 4, 3, 40)] * 2 + [(2, 4, 1, 64)] * 4
