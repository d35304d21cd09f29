"""Paged caches of keys and values, and attention of new tokens over them.

A *pool* is a tensor (pages, page_size, kv_heads, dim) that holds one key or value set of one layer.  Position x of sequence s is row
``x % page_size`` of page ``tables[s, x // page_size]``; ``lengths[s]`` tokens of a sequence are in the cache, the new ones included, and ``counts[s]``
(default: all) of a call's rows are there, the rest being padding: row t is at position ``lengths[s] - counts[s] + t``.  ``tables``, ``lengths`` and ``counts`` are int32
tensors on the GPU, read by the kernels alone: a table entry outside 0 .. pages - 1, like a position beyond the table, is a place that is not there, of which
nothing is attended to or written. 
"""
from __future__ import annotations

import heapq
from dataclasses import dataclass
from typing import Sequence

import torch
from torch import Tensor

from . import _native


def paged_attn(q: Tensor, k_pages: Tensor, v_pages: Tensor, tables: Tensor, lengths: Tensor, counts: Tensor | None = None, *, scale: float | None = None,
               max_length: int | None = None) -> Tensor:
    """Dense causal attention of a chunk of new tokens over a paged cache that holds them already: q (b, n, h, d) -> (b, n, h, d).

    Query head h reads key/value head ``h // (h_q / h_kv)``.  q and the pools share one dtype, bfloat16 or float16; the pools have d channels, or more if
    those beyond d are zero.  Softmax weights are rounded to that dtype for their product with the values; sums are float32.  Rows that attend to nothing, padding among them,
    are zero.  ``max_length``: no sequence is longer (it saves launching work for what the tables could name; a wrong value costs time, not correctness).
    """
    return _native.torch_ext().paged_attend(q, [k_pages], [v_pages], tables, lengths, counts, 1, 1, scale, max_length)


def paged_two_simplicial_attn(q: Tensor, keys: tuple[Tensor, Tensor], values: tuple[Tensor, Tensor], tables: Tensor, lengths: Tensor, counts: Tensor | None = None, *,
                              w1=512, w2=32, scale: float | None = None, max_length: int | None = None) -> Tensor:
    """:func:`sliding_two_simplicial_attn` for a chunk of new tokens over a paged cache that holds them already: the row at position p attends to the pairs
    ``p - w1 < j <= p``, ``p - w2 < k <= p``.  Arguments as in :func:`paged_attn`, two key and two value pools."""
    if len(keys) != 2 or len(values) != 2:
        raise AssertionError('two key sets and two value sets are required')
    return _native.torch_ext().paged_attend(q, list(keys), list(values), tables, lengths, counts, int(w1), int(w2), scale, max_length)


def paged_append(pages: Sequence[Tensor], rows: Sequence[Tensor], tables: Tensor, lengths: Tensor, counts: Tensor | None = None) -> None:
    """Writes new rows (b, n, kv_heads, d) into the pages of up to four pools that share one geometry.  The rows are bfloat16, float16 or float32 and rounded
    to the pools' dtype; channels of the pools beyond d become zero in the written rows."""
    _native.torch_ext().paged_append(list(pages), list(rows), tables, lengths, counts)


def copy_pages(pages: Sequence[Tensor], pairs) -> None:
    """In every pool, page ``pairs[i][0]`` to page ``pairs[i][1]`` for all i.  ``pairs``: a (count, 2) integer tensor in host memory, or a sequence of pairs.  Pages that
    do not exist are refused, and so is a page that is written twice or written and read (the pairs run in no order)."""
    if not isinstance(pairs, Tensor):
        pairs = torch.tensor(list(pairs), dtype=torch.int64).reshape(-1, 2)
    _native.torch_ext().copy_pages(list(pages), pairs)


class OutOfPages(RuntimeError):
    """A cache has too few free pages for a call; the call has changed nothing."""


@dataclass(frozen=True)
class PagedBatch:
    """Where the rows of a call go: what :func:`paged_append` and the attention functions take for the sequences of one call, in its order."""
    tables: Tensor          # (b, entries) int32
    lengths: Tensor         # (b,) int32, the new tokens included
    counts: Tensor          # (b,) int32 new tokens
    max_length: int


class PagedCache:
    """Keys and values of many sequences for all layers of a model, in pages that sequences take, share and give back.

    ``layers``: for each layer ``(sets, kv_heads, dim_head)``; ``keys[layer]`` and ``values[layer]`` are tuples of ``sets`` pools.  One table of pages serves all
    layers.  The pages of a forked sequence are shared until one of the sharers writes into the last, partly filled one, which is copied then.  Which page
    belongs to whom is kept on the host, so running out of pages is an exception and nothing here waits for the GPU; copies and uploads are queued on the
    current stream, and calls that use the cache on another one have to be ordered by the caller.
    """

    def __init__(self, layers: Sequence[tuple[int, int, int]], *, pages: int, page_size: int = 64, dtype: torch.dtype = torch.bfloat16, device='cuda'):
        if pages < 1 or page_size < 1:
            raise ValueError('a cache needs pages, and pages rows')
        if dtype not in (torch.bfloat16, torch.float16):
            raise TypeError(f'unsupported dtype {dtype}')
        # (as a device of its own: 'cuda' alone is whichever is current)
        self.page_size, self.pages, self.device = page_size, pages, torch.empty(0, device=device).device
        self.keys, self.values = [], []
        for sets, kv_heads, dim in layers:
            # (channels in whole 16-byte pieces; the rows are written before they are read, so nothing needs clearing)
            shape = (pages, page_size, kv_heads, -(-dim // 8) * 8)
            self.keys.append(tuple(torch.empty(shape, dtype=dtype, device=device) for _ in range(sets)))
            self.values.append(tuple(torch.empty(shape, dtype=dtype, device=device) for _ in range(sets)))
        self._free = list(range(pages))           # a heap: the lowest free page is taken first
        self._shares = [0] * pages
        self._tables: dict[int, list[int]] = {}
        self._lengths: dict[int, int] = {}
        self._next = 0

    # ---- what is in the cache
    @property
    def pools(self) -> list[Tensor]:
        return [pool for keys, values in zip(self.keys, self.values) for pool in (*keys, *values)]

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def length(self, sequence: int) -> int:
        return self._lengths[self._known(sequence)]

    def table(self, sequence: int) -> list[int]:
        return list(self._tables[self._known(sequence)])

    def _known(self, sequence):
        if sequence not in self._tables:
            raise KeyError(f'no sequence {sequence} in this cache')
        return sequence

    # ---- sequences come, grow and go
    def new(self) -> int:
        """An empty sequence; its name."""
        name, self._next = self._next, self._next + 1
        self._tables[name], self._lengths[name] = [], 0
        return name

    def fork(self, sequence: int) -> int:
        """A new sequence with the tokens of ``sequence``, on the same pages."""
        pages = self._tables[self._known(sequence)]
        name = self.new()
        for page in pages:
            self._shares[page] += 1
        self._tables[name], self._lengths[name] = list(pages), self._lengths[sequence]
        return name

    def free(self, *sequences: int) -> None:
        """Forgets sequences; pages that no other one shares can be taken again."""
        if len(set(sequences)) < len(sequences):
            raise ValueError('a sequence is freed twice')
        for sequence in sequences:
            self._known(sequence)
        for sequence in sequences:
            self._give_back(self._tables.pop(sequence))
            del self._lengths[sequence]

    def truncate(self, sequence: int, length: int) -> None:
        """Forgets the tokens from ``length`` on (guesses that were not accepted)."""
        if not 0 <= length <= self._lengths[self._known(sequence)]:
            raise ValueError(f'sequence {sequence} has {self._lengths[sequence]} tokens, not {length}')
        keep = -(-length // self.page_size)
        table = self._tables[sequence]
        self._give_back(table[keep:])
        del table[keep:]
        self._lengths[sequence] = length

    def _give_back(self, pages):
        for page in pages:
            self._shares[page] -= 1
            if self._shares[page] == 0:
                heapq.heappush(self._free, page)

    def _take(self):
        page = heapq.heappop(self._free)
        self._shares[page] = 1
        return page

    def extend(self, sequences: Sequence[int], counts: Sequence[int] | int) -> PagedBatch:
        """Room for ``counts`` new tokens in each of ``sequences``: takes pages, makes the ones that will be written the sequences' own, and returns where the
        rows of the call go.  Raises :class:`OutOfPages` before anything has changed."""
        counts = [counts] * len(sequences) if isinstance(counts, int) else list(counts)
        if len(counts) != len(sequences) or len(set(sequences)) < len(sequences) or any(c < 0 for c in counts):
            raise ValueError('a call extends different sequences, each by a number of tokens')
        needed, shares = 0, {}
        for sequence, count in zip(sequences, counts):
            table, length = self._tables[self._known(sequence)], self._lengths[sequence]
            needed += -(-(length + count) // self.page_size) - len(table)
            if count and length % self.page_size:
                last = table[-1]
                left = shares.setdefault(last, self._shares[last])
                if left > 1:                      # (of the sharers of a page the last one to write keeps it)
                    needed += 1
                    shares[last] = left - 1
        if needed > len(self._free):
            raise OutOfPages(f'{needed} pages are needed, {len(self._free)} of {self.pages} are free')
        copies = []
        for sequence, count in zip(sequences, counts):
            table, length = self._tables[sequence], self._lengths[sequence]
            if count and length % self.page_size and self._shares[table[-1]] > 1:
                old = table[-1]
                table[-1] = self._take()
                self._shares[old] -= 1
                copies.append((old, table[-1]))
            for _ in range(-(-(length + count) // self.page_size) - len(table)):
                table.append(self._take())
            self._lengths[sequence] = length + count
        if copies:
            copy_pages(self.pools, copies)
        return self._batch(sequences, counts)

    def _batch(self, sequences, counts):
        lengths = [self._lengths[s] for s in sequences]
        width = max((len(self._tables[s]) for s in sequences), default=0)
        rows = [self._tables[s] + [-1] * (width - len(self._tables[s])) + [length, count] for s, length, count in zip(sequences, lengths, counts)]
        flat = torch.tensor(rows, dtype=torch.int32).view(len(rows), width + 2)
        on_gpu = (flat.pin_memory() if flat.numel() else flat).to(self.device, non_blocking=True)
        return PagedBatch(on_gpu[:, :width], on_gpu[:, width].contiguous(), on_gpu[:, width + 1].contiguous(), max(lengths, default=0))

    def compact(self) -> int:
        """Moves the pages in use to the front of the pools; returns how many were moved.  Batches that :meth:`extend` returned before name places that are no longer
        the sequences'."""
        used = self.pages - len(self._free)
        holes = sorted(page for page in self._free if page < used)
        strays = [page for page in range(used, self.pages) if self._shares[page]]
        if not strays:
            return 0
        copy_pages(self.pools, list(zip(strays, holes)))
        to = dict(zip(strays, holes))
        for table in self._tables.values():
            table[:] = [to.get(page, page) for page in table]
        for old, new in to.items():
            self._shares[new], self._shares[old] = self._shares[old], 0
        self._free = list(range(used, self.pages))
        return len(strays)
