"""Paged caches of keys and values, and attention of new tokens over them.

A *pool* is a tensor (pages, page_size, kv_heads, dim) that holds one key or value set of one layer.  Position x of sequence s is row
``x % page_size`` of page ``tables[s, x // page_size]``; ``lengths[s]`` tokens of a sequence are in the cache, the new ones included, and ``counts[s]``
(default: all) of a call's rows are there, the rest being padding: row t is at position ``lengths[s] - counts[s] + t``.  ``tables``, ``lengths`` and ``counts`` are int32
tensors on the GPU, read by the kernels alone: a table entry outside 0 .. pages - 1, like a position beyond the table, is a place that is not there, of which
nothing is attended to or written. 
"""
from __future__ import annotations

from typing import Sequence

import torch
from torch import Tensor

from . import _native


def paged_attn(q: Tensor, k_pages: Tensor, v_pages: Tensor, tables: Tensor, lengths: Tensor, counts: Tensor | None = None, *, scale: float | None = None,
               max_length: int | None = None) -> Tensor:
    """Dense causal attention of a chunk of new tokens over a paged cache that holds them already: q (b, n, h, d) -> (b, n, h, d).

    Query head h reads key/value head ``h // (h_q / h_kv)``.  q and the pools share one dtype, bfloat16 or float16; the pools have d channels, or more if
    those beyond d are zero.  Rows that attend to nothing, padding among them, are zero.  ``max_length``: no sequence is longer (it saves launching work for what the
    tables could name; a wrong value costs time, not correctness).
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
