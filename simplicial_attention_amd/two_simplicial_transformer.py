"""Decoder stack that interleaves ordinary causal attention with sliding-window 2-simplicial
attention, and a byte-level language-model wrapper around it.

Counterparts of simplicial_attention/two_simplicial_transformer.py:24-141 (``Attention``,
``FeedForward``, ``TwoSimplicialTransformer``) and of the ``TwoSimplicialLM`` class of
train.py:64-135 in the reference, with the same constructor arguments and the same
parameter names, so that a reference ``state_dict`` loads unchanged.  The ordinary layers
are library calls (``scaled_dot_product_attention``, ``Linear``); every
``two_simplicial_attn_every``-th layer is the MI355X module of this package.
"""
from __future__ import annotations

import torch
import torch.nn.functional as F
from torch import nn

from .linear import apply_linear
from .paged import PagedCache, paged_append, paged_attn
from .sampling import sample_tokens
from .two_simplicial_attention import SlidingWindowTwoSimplicialMHA


class Attention(nn.Module):
    """Pre-normed causal attention with grouped key/value heads
    (two_simplicial_transformer.py:24-65)."""

    def __init__(self, dim, dim_head=64, heads=8, key_value_heads=8):
        super().__init__()
        if heads % key_value_heads:
            raise AssertionError('heads must be a multiple of key_value_heads')
        self.heads, self.key_value_heads, self.dim_head = heads, key_value_heads, dim_head
        self.prenorm = nn.RMSNorm(dim)
        self.to_q = nn.Linear(dim, heads * dim_head, bias=False)
        self.to_kv = nn.Linear(dim, 2 * key_value_heads * dim_head, bias=False)
        self.to_out = nn.Linear(heads * dim_head, dim, bias=False)

    def forward(self, x):
        b, n, _ = x.shape
        x = self.prenorm(x)
        if torch.jit.is_scripting():      # (a scripted module takes its own submodules only)
            q, kv = self.to_q(x), self.to_kv(x)
        else:
            q, kv = apply_linear(self.to_q, x), apply_linear(self.to_kv, x)
        q = q.view(b, n, self.heads, self.dim_head).transpose(1, 2)
        # channel order of the fused projection: (key | value, head, d)
        kv = kv.view(b, n, 2, self.key_value_heads, self.dim_head)
        k, v = kv[:, :, 0].transpose(1, 2), kv[:, :, 1].transpose(1, 2)
        out = F.scaled_dot_product_attention(q, k, v, is_causal=True, enable_gqa=self.heads != self.key_value_heads)
        out = out.transpose(1, 2).reshape(b, n, self.heads * self.dim_head)
        if torch.jit.is_scripting():
            return self.to_out(out)
        return apply_linear(self.to_out, out)


    @torch.no_grad()
    @torch.jit.unused
    def forward_cached(self, x, keys, values, batch):
        """``forward`` for new tokens (b, n, dim) behind those in a paged cache: the layer's key and value pool (tuples of one), and where the rows go.  Queries, keys and
        values are rounded to the pools' dtype."""
        b, n, _ = x.shape
        x = self.prenorm(x)
        q = self.to_q(x).view(b, n, self.heads, self.dim_head)
        k, v = self.to_kv(x).view(b, n, 2, self.key_value_heads, self.dim_head).unbind(2)
        at = (batch.tables, batch.lengths, batch.counts)
        paged_append((*keys, *values), (k, v), *at)
        out = paged_attn(q.to(keys[0].dtype), *keys, *values, *at, max_length=batch.max_length)
        return self.to_out(out.to(x.dtype).reshape(b, n, self.heads * self.dim_head))


class _Layers(nn.Sequential):
    """``nn.Sequential`` whose plain linear layers go through ``apply_linear``."""

    def forward(self, x):
        if torch.jit.is_scripting():
            for layer in self:
                x = layer(x)
        else:
            for layer in self:
                x = apply_linear(layer, x)
        return x


def FeedForward(dim, expansion=4.):
    """RMSNorm -> Linear -> GELU -> Linear (two_simplicial_transformer.py:69-76)."""
    inner = int(dim * expansion)
    return _Layers(nn.RMSNorm(dim), nn.Linear(dim, inner), nn.GELU(), nn.Linear(inner, dim))


class TwoSimplicialTransformer(nn.Module):
    def __init__(self, dim, *, depth, heads=8, key_value_heads=4, dim_head=64, ff_expansion=4.,
                 two_simplicial_attn_every=4, attn_kwargs: dict | None = None,
                 two_simplicial_attn_kwargs: dict | None = None, final_norm=True):
        super().__init__()
        attn_kwargs = {} if attn_kwargs is None else attn_kwargs
        if two_simplicial_attn_kwargs is None:
            two_simplicial_attn_kwargs = dict(w1=512, w2=32, qk_rmsnorm=True)
        blocks = []
        for index in range(1, depth + 1):
            common = dict(dim=dim, heads=heads, key_value_heads=key_value_heads, dim_head=dim_head)
            if index % two_simplicial_attn_every == 0:
                attn = SlidingWindowTwoSimplicialMHA(prenorm=True, **common, **two_simplicial_attn_kwargs)
            else:
                attn = Attention(**common, **attn_kwargs)
            blocks.append(nn.ModuleList([attn, FeedForward(dim, ff_expansion)]))
        self.layers = nn.ModuleList(blocks)
        self.norm = nn.RMSNorm(dim) if final_norm else nn.Identity()

    def forward(self, x):
        for attn, ff in self.layers:
            x = x + attn(x)
            x = x + ff(x)
        return self.norm(x)

    def cache(self, pages, page_size=64, dtype=None) -> PagedCache:
        """An empty cache for this stack's layers, on its device (in its dtype, or bfloat16 for float32 weights)."""
        weight = next(self.parameters())
        if dtype is None:
            dtype = weight.dtype if weight.dtype in (torch.bfloat16, torch.float16) else torch.bfloat16
        layers = []
        for attn, _ in self.layers:
            if isinstance(attn, Attention):
                layers.append((1, attn.key_value_heads, attn.dim_head))
            else:
                layers.append((2, attn.key_value_heads, max(attn.split_dims[0] // attn.heads, attn.split_dims[2] // (2 * attn.key_value_heads))))
        return PagedCache(layers, pages=pages, page_size=page_size, dtype=dtype, device=weight.device)

    @torch.no_grad()
    def forward_cached(self, x, cache, batch):
        """The stack for new tokens (b, n, dim) whose places ``batch = cache.extend(...)`` has made; rows beyond ``batch.counts`` are padding.  Queries, keys and values are
        rounded to the cache's dtype."""
        for (attn, ff), keys, values in zip(self.layers, cache.keys, cache.values):
            x = x + attn.forward_cached(x, keys, values, batch)
            x = x + ff(x)
        return self.norm(x)


class TwoSimplicialLM(nn.Module):
    """Token + learned position embedding, the stack above, and a linear read-out
    (train.py:64-135).  ``generate`` answers prompts from a paged cache (the reference recomputes the sequence for every token)."""

    def __init__(self, *, num_tokens, dim, depth, max_seq_len=512, dim_head=64, heads=8,
                 two_simplicial_attn_every=4, transformer_kwargs: dict | None = None):
        super().__init__()
        self.token_emb = nn.Embedding(num_tokens, dim)
        self.pos_emb = nn.Embedding(max_seq_len, dim)
        self.transformer = TwoSimplicialTransformer(dim=dim, depth=depth, dim_head=dim_head, heads=heads,
                                                    two_simplicial_attn_every=two_simplicial_attn_every,
                                                    **(transformer_kwargs or {}))
        self.to_logits = nn.Linear(dim, num_tokens, bias=False)

    def forward(self, x, return_loss=False):
        target = None
        if return_loss:
            x, target = x[:, :-1], x[:, 1:]
        positions = torch.arange(x.shape[-1], device=x.device)
        hidden = self.transformer(self.token_emb(x) + self.pos_emb(positions))
        logits = apply_linear(self.to_logits, hidden)
        if target is None:
            return logits
        return F.cross_entropy(logits.flatten(0, 1).float(), target.flatten())

    @torch.no_grad()
    def logits_cached(self, x, cache, batch, rows=None):
        """Logits of new tokens (b, n) whose places ``batch = cache.extend(...)`` has made; ``rows`` (b,): of that row of each sequence alone, (b, num_tokens).
        Sequences longer than the table of positions are refused."""
        if batch.max_length > self.pos_emb.num_embeddings:
            raise ValueError(f'a sequence of {batch.max_length} tokens, positions reach {self.pos_emb.num_embeddings}')
        at = (batch.lengths - batch.counts)[:, None] + torch.arange(x.shape[1], device=x.device)
        # (padding reads some row of the table)
        hidden = self.transformer.forward_cached(self.token_emb(x) + self.pos_emb(at.clamp(0, self.pos_emb.num_embeddings - 1)), cache, batch)
        if rows is not None:
            hidden = hidden[torch.arange(len(x), device=x.device), rows]
        return self.to_logits(hidden)

    @torch.no_grad()
    def generate(self, prompts, steps, *, lengths=None, samples=1, temperature=1., top_k=0, top_p=1., min_p=0., generator=None, chunk=512, page_size=64, dtype=None):
        """``steps`` tokens behind every prompt: prompts (b, n) -> (b, samples, steps) tokens and their log-probabilities.

        ``lengths``: tokens of each prompt (host numbers), the others of its row being padding; by default all are prompt.  Prompts are read in chunks of ``chunk`` tokens into a
        paged cache, once for all of a prompt's ``samples``, which share its pages.  Tokens are drawn by :func:`sample_tokens` with uniform
        numbers from ``generator``.

        ``dtype``: of the cache, bfloat16 or float16 (by default the weights', bfloat16 for float32 ones).  Queries, keys and values are rounded to it, those of float32 weights
        to 8 or 11 bits, of which ``forward`` rounds the 2-simplicial layers' alone (to bfloat16).
        """
        b, n = prompts.shape
        lengths = [n] * b if lengths is None else [int(length) for length in lengths]
        if len(lengths) != b or steps < 1 or samples < 1 or chunk < 1 or not all(1 <= length <= n for length in lengths):
            raise ValueError('every prompt needs 1 to n tokens, and steps, samples and chunk are at least 1')
        if max(lengths) + steps - 1 > self.pos_emb.num_embeddings:
            raise ValueError(f'{max(lengths)} + {steps} tokens, positions reach {self.pos_emb.num_embeddings}')
        shared = sum(-(-length // page_size) for length in lengths)
        own = samples * sum(-(-(length + steps) // page_size) - length // page_size for length in lengths)
        cache = self.transformer.cache(shared + own, page_size, dtype)
        sequences = [cache.new() for _ in range(b)]
        first = None
        for start in range(0, max(lengths), chunk):
            counts = [min(max(length - start, 0), chunk) for length in lengths]
            part = prompts[:, start:start + max(counts)]
            ends = torch.tensor([min(max(length - 1 - start, 0), part.shape[1] - 1) for length in lengths], device=prompts.device)
            logits = self.logits_cached(part, cache, cache.extend(sequences, counts), ends)
            ended = torch.tensor([start < length <= start + chunk for length in lengths], device=prompts.device)
            first = logits if first is None else torch.where(ended[:, None], logits, first)
        sequences = [s for prompt in sequences for s in (prompt, *(cache.fork(prompt) for _ in range(samples - 1)))]
        logits = first.repeat_interleave(samples, 0)
        tokens, logprobs = [], []
        for step in range(steps):
            noise = torch.rand(logits.shape, generator=generator, device=logits.device)
            token, logprob = sample_tokens(logits, noise, temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p)
            tokens.append(token)
            logprobs.append(logprob)
            if step + 1 < steps:
                logits = self.logits_cached(token[:, None], cache, cache.extend(sequences, 1))[:, 0]
        return torch.stack(tokens, 1).view(b, samples, steps), torch.stack(logprobs, 1).view(b, samples, steps)
