"""Linear layers whose weight gradient runs on this package's kernel where that is the faster one."""
from __future__ import annotations

import torch
import torch.nn.functional as F
from torch import Tensor, nn
from torch.nn.modules import module as _module
from torch.utils._device import DeviceContext

from . import _native


# what a call of a module goes through, as torch has it
_CALL, _CALL_IMPL = nn.Module.__call__, nn.Module._call_impl
_FORWARD, _LINEAR = nn.Linear.forward, F.linear


def modes():
    """Someone sees torch's operators or functions (the kernels of this package are none)."""
    return torch._C._len_torch_dispatch_stack() or torch._C._len_torch_function_stack()


def modes_but_devices():
    """The same, but for a default device (``torch.set_default_device``, ``with torch.device(...)``), which is a mode that changes the calls of factories alone."""
    return torch._C._len_torch_dispatch_stack() or any(type(torch._C._get_function_stack_at(i)) is not DeviceContext for i in range(torch._C._len_torch_function_stack()))


def all_watched():
    """Someone sees the calls of all modules, or has changed what they are."""
    return bool(nn.Module.__call__ is not _CALL or nn.Module._call_impl is not _CALL_IMPL or _module._global_forward_hooks or _module._global_forward_pre_hooks
                or _module._global_backward_hooks or _module._global_backward_pre_hooks)


def watched(module):
    """Someone else sees the calls of this module, or has changed what it is."""
    return bool(module._compiled_call_impl is not None or module._forward_hooks or module._forward_pre_hooks or module._backward_hooks or module._backward_pre_hooks
                or 'forward' in module.__dict__)


def _watched(layer):
    return (nn.Linear.forward is not _FORWARD or nn.Linear.__call__ is not _CALL or nn.Linear._call_impl is not _CALL_IMPL or F.linear is not _LINEAR
            or watched(layer) or all_watched())


def _faster(rows, out_features, in_features):
    # Measured against the library (us, ours and the library's): 8192 rows, 2048 x 512: 37, 55; 512 x 512: 24, 52; 2048 x 1024: 54, 68;
    # 16384 rows, 2048 x 512: 53, 104; 65536 rows, 2048 x 1024: 308, 368.  The library does not split the rows: with fewer of them
    # (4096 rows, 2048 x 1024: 38, 37) or larger results (65536 rows, 3072 x 1024: 578, 477) it is as fast or faster.
    return rows >= 8192 and out_features % 128 == 0 and in_features % 128 == 0 and out_features * in_features <= 2048 * 1024


def apply_linear(layer, x):
    """``layer(x)``; plain bf16 ``nn.Linear`` layers under training take the node with the kernel of their own."""
    # (torch.fx hands over proxies: the type comes first)
    if (type(x) is not Tensor or type(layer) is not nn.Linear or torch.compiler.is_compiling() or torch.jit.is_tracing()
            or not x.is_cuda or not torch.is_grad_enabled()):
        return layer(x)
    weight, bias = layer.weight, layer.bias
    if (type(weight) is not nn.Parameter or type(bias) not in (nn.Parameter, type(None))
            or x.dtype is not torch.bfloat16 or weight.dtype is not torch.bfloat16 or (bias is not None and bias.dtype is not torch.bfloat16)
            or x.device != weight.device or x.dim() < 2 or x.shape[-1] != weight.shape[1]
            or not _faster(x.numel() // x.shape[-1] if x.shape[-1] else 0, *weight.shape)
            or torch.is_autocast_enabled() or modes() or _watched(layer)):
        return layer(x)
    return _native.torch_ext().linear(x, weight, bias)
