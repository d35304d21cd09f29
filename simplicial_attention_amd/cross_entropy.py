"""Softmax cross entropy of a read-out layer over a large vocabulary, without its logits."""
from __future__ import annotations

from torch import Tensor

from . import _native

_REDUCTIONS = ('none', 'mean', 'sum')


def linear_cross_entropy(hidden: Tensor, weight: Tensor, targets: Tensor, *, ignore_index: int = -100, reduction: str = 'mean') -> Tensor:
    """``cross_entropy(hidden @ weight.T, targets)`` in float32, differentiable in ``hidden`` (..., dim) and ``weight`` (vocab, dim); ``targets`` (...) are int64 or int32.

    The logits are never kept: the forward leaves a maximum and a sum of each row, the backward forms them again in pieces of the vocabulary (up to 256 MiB of their
    gradients at a time, rounded to the operands' dtype, bfloat16 or float16).  While it runs the forward takes 8 bytes for every 64 or 128 logits of a row (512 MiB for 65536
    rows over 131072 tokens).  Operands whose rows are not aligned to 16 bytes, or whose channels are no multiple of 8, are copied, and the copies kept for the backward.

    Rows whose target is ``ignore_index`` have no loss and no gradient and add nothing to the weight's, whatever they hold.  Any other target outside the vocabulary makes the results NaN.
    ``reduction``: 'mean' over the rows that count (NaN without any, its gradients zero), 'sum', or 'none' for a loss per row, whose gradients may weigh the rows as far apart as
    float32 goes: a row of ``hidden``'s does not depend on the others' weights (``weight``'s, in float16, has of each row an error of up to 2**-35 of the largest weight times the row).
    Recorders (``torch.jit.trace``, ``make_fx``) are refused: they do not see the kernels.
    """
    if reduction not in _REDUCTIONS:
        raise ValueError(f"reduction must be 'none', 'mean' or 'sum', got {reduction!r}")
    return _native.torch_ext().linear_cross_entropy(hidden, weight, targets, ignore_index, _REDUCTIONS.index(reduction))
