"""The residual's addition and the RMSNorm behind it in one pass over the rows, with gradients, and with an output in 8 bits."""
from __future__ import annotations

import torch
import torch.nn.functional as F
from torch import Tensor, nn

from . import _native
from .linear import all_watched, modes_but_devices, watched


def add_rms_norm(x: Tensor, residual: Tensor | None = None, weight: Tensor | None = None, eps: float | None = None) -> tuple[Tensor, Tensor]:
    """``total = x + residual`` and ``normed = rms_norm(total, weight, eps)`` over the last dimension: ``(normed, total)``, both differentiable.

    What ``x = x + attn(x); y = norm(x)`` of a pre-normed stack computes, to the bit but for the order of the sums: total is rounded to its dtype (the
    residual's: that of x, or float32 for a residual stream in 32 bits) and normalised as rounded, with float32 sums; normed has the dtype of x.  Without a residual total is x itself.
    ``weight`` (dim,) may have a dtype of its own; ``eps=None`` is float32's, as in ``torch.nn.RMSNorm`` (which takes float32's for narrower inputs too).  bfloat16, float16 and float32 tensors
    on the GPU of any strides, rows of up to 16384 channels.  Recorders (``torch.jit.trace``, ``make_fx``) are refused: they do not see the kernel.
    """
    return _native.torch_ext().add_rms_norm(x, residual, weight, eps)


def add_rms_norm_8bit(x: Tensor, residual: Tensor | None = None, weight: Tensor | None = None, eps: float | None = None, *,
                      group: int | None = None) -> tuple[Tensor, Tensor, Tensor]:
    """:func:`add_rms_norm` with its first output as operands of an 8-bit product: ``(values, scales, total)``, for inference.

    ``values`` are float8_e4m3fn, ``scales`` float32, one per row (..., 1), or with ``group`` 32, 64 or 128 one per so many channels (..., ceil(dim / group)):
    scale = max(amax / 448, 2**-126) over the row or group, value = the nearest e4m3 to normed / scale (which is not rounded to x's dtype in between).  A group that holds a value
    that is not a number has no number as its scale.
    """
    return _native.torch_ext().add_rms_norm_8bit(x, residual, weight, eps, 0 if group is None else group)


_FORWARD, _RMS_NORM = nn.RMSNorm.forward, F.rms_norm
_PLAIN = (Tensor, nn.Parameter)


def _covered(norm):
    """What this module computes is the kernel's to compute, and nobody sees its calls."""
    return (type(norm) is nn.RMSNorm and type(norm.weight) in _PLAIN and nn.RMSNorm.forward is _FORWARD and nn.RMSNorm.__call__ is nn.Module.__call__ and F.rms_norm is _RMS_NORM
            and not (modes_but_devices() or all_watched() or watched(norm)))


def norm_behind(norm, x: Tensor, residual: Tensor | None) -> tuple[Tensor, Tensor]:
    """``total = x + residual`` (x alone without one) and ``norm(total)`` of an ``nn.RMSNorm`` module: ``(normed, total)``.  Modules and tensors that the kernel does not cover, and modules
    whose calls someone sees (hooks, tracers, modes), go through torch."""
    # (torch.fx hands over proxies: the type comes first)
    if (torch.compiler.is_compiling() or torch.jit.is_tracing() or type(x) not in _PLAIN or not _covered(norm) or not x.is_cuda or norm.normalized_shape != (x.shape[-1],)
            or torch.is_autocast_enabled()
            or norm.weight.dtype != x.dtype or (residual is not None and (type(residual) not in _PLAIN or residual.dtype != x.dtype))
            or not _native.torch_ext().norm_covers(x, residual, norm.weight)):
        total = x if residual is None else residual + x
        return norm(total), total
    return add_rms_norm(x, residual, norm.weight, norm.eps)
