"""Next tokens from logits and given random numbers."""
from __future__ import annotations

import math

import torch
from torch import Tensor

from . import _native


def sample_tokens(logits: Tensor, noise: Tensor, *, temperature=1., top_k=0, top_p=1., min_p=0.) -> tuple[Tensor, Tensor]:
    """One token per row of ``logits`` (..., vocab): ``(tokens, logprobs)`` of shape (...), int64 and float32.

    The tokens of a row are ordered by (logit descending, index ascending) and weighed by p = softmax(logits / temperature).  A token is
    kept if its rank is below ``top_k`` (0: any), the mass in front of it below ``top_p`` (1: any) and p at least ``min_p`` times the largest; the
    first always is.  The result is the kept token with the largest ``logits / temperature - log(-log(noise))``: a draw from p among the kept tokens
    where ``noise`` (float32, the shape of ``logits``) is uniform on [0, 1).  ``temperature`` 0 takes the first token of the order.  ``logprobs`` are the tokens'
    logarithms under softmax(logits).  A logit that is not a number counts as -inf; a row without any other gives token -1 and -inf.

    Every parameter is a number, or a tensor with one value per row (float32; ``top_k`` int32).  Numbers have to be finite and not negative.  Tensors are read by the kernels alone: a
    negative temperature is taken as 0, an infinite one weighs all tokens above -inf alike, and a value that is not a number leaves its row the first token.
    """
    given = dict(temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p)
    tensors = {name: value if isinstance(value, Tensor) else None for name, value in given.items()}
    numbers = {name: default if isinstance(value, Tensor) else value for (name, value), default in zip(given.items(), (1., 0, 1., 0.))}
    for name, value in numbers.items():
        if not math.isfinite(value) or value < 0:
            raise ValueError(f'{name} must be finite and not negative, got {value}')
    return _native.torch_ext().sample_tokens(logits, noise, *tensors.values(), float(numbers['temperature']), int(numbers['top_k']), float(numbers['top_p']),
                                             float(numbers['min_p']))
