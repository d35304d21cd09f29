"""A fused stack whose modules' calls, or operators, someone watches or has replaced runs as the separate calls."""
import pytest
import torch
import torch.nn.functional as F
from torch import nn
from torch.overrides import TorchFunctionMode
from torch.utils._python_dispatch import TorchDispatchMode

from simplicial_attention_amd.two_simplicial_transformer import Attention, TwoSimplicialLM, TwoSimplicialTransformer

DEVICES = ['cpu', pytest.param('cuda', marks=pytest.mark.gpu)]


def stack(fused, device='cpu', dtype=torch.float32):
    torch.manual_seed(0)
    return TwoSimplicialTransformer(64, depth=3, heads=2, key_value_heads=2, dim_head=32, two_simplicial_attn_every=4, fused=fused).to(device, dtype)


def language_model(fused, device):
    torch.manual_seed(0)
    return TwoSimplicialLM(num_tokens=50, dim=64, depth=2, heads=2, dim_head=32, two_simplicial_attn_every=4, transformer_kwargs=dict(key_value_heads=2), fused=fused).to(device, torch.bfloat16)


def rows(device='cpu'):
    return torch.randn(2, 9, 64, generator=torch.Generator().manual_seed(1)).to(device)


def close(a, b):
    # (norms that are not replaced add up 64 squares in another order: some last places of 2^-24 in each of seven norms; what is replaced is larger by a factor)
    return torch.equal(a, b) if not a.is_cuda else float(((a - b).norm() / a.norm()).detach()) < 2. ** -18


@pytest.mark.parametrize('device', DEVICES)
def test_global_hooks_see_every_module(device):
    x, seen = rows(device), []
    for fused in (False, True):
        modules = []
        handle = nn.modules.module.register_module_forward_hook(lambda module, *_: modules.append(type(module).__name__))
        try:
            out = stack(fused, device)(x)
        finally:
            handle.remove()
        seen.append((modules, out))
    assert seen[0][0] == seen[1][0] and torch.equal(seen[0][1], seen[1][1])


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('mode', [TorchDispatchMode, TorchFunctionMode])
def test_modes_see_every_operator(device, mode):
    class Seen(mode):
        def __init__(self):
            super().__init__()
            self.calls = []

        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            self.calls.append(str(func))
            return func(*args, **(kwargs or {}))

        def __torch_function__(self, func, types, args=(), kwargs=None):
            self.calls.append(getattr(func, '__name__', str(func)))
            return func(*args, **(kwargs or {}))
    tokens = torch.arange(16, device=device).view(2, 8)
    seen = []
    for fused in (False, True):
        lm = language_model(fused, device)
        with Seen() as calls:
            loss = lm(tokens, return_loss=True)
        seen.append((calls.calls, loss.detach()))
    assert seen[0][0] == seen[1][0] and torch.equal(seen[0][1], seen[1][1])


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('which', ['prenorm', 'ff_norm', 'norm', 'attn', 'ff'])
def test_replaced_forwards_are_called(device, which):
    x, outs = rows(device), []
    for fused in (False, True):
        t = stack(fused, device)
        attn, ff = t.layers[1]
        module = {'prenorm': attn.prenorm, 'ff_norm': ff[0], 'norm': t.norm, 'attn': attn, 'ff': ff}[which]
        module.forward = lambda x: 3 * x
        outs.append(t(x))
    assert close(*outs)


@pytest.mark.parametrize('device', DEVICES)
def test_replaced_classes_and_functions_are_called(device, monkeypatch):
    x = rows(device)
    separate, fused = stack(False, device), stack(True, device)
    for owner, name, other in ((nn.RMSNorm, 'forward', lambda self, x: 2 * x), (Attention, 'forward', lambda self, x: x.sin()), (F, 'rms_norm', lambda x, *_: 4 * x),
                               (nn.RMSNorm, '__call__', lambda self, x: 5 * x), (Attention, '__call__', lambda self, x: x.cos())):
        with monkeypatch.context() as patch:
            patch.setattr(owner, name, other)
            assert torch.equal(fused(x), separate(x)), name


def test_symbolic_traces_of_a_fused_stack():
    x, t = rows(), stack(True)
    assert torch.equal(torch.fx.symbolic_trace(t)(x), t(x))


@pytest.mark.gpu
def test_compiled_norms_are_called():
    x, outs = rows('cuda'), []
    for fused in (False, True):
        t, calls = stack(fused, 'cuda'), []
        t.norm._compiled_call_impl = lambda x: calls.append(1) or 2 * x
        outs.append(t(x))
        assert calls == [1]
    assert close(*outs)


def test_a_fused_stack_makes_no_modules(monkeypatch):
    x, t = rows(), stack(True)
    want = stack(False)(x)
    monkeypatch.setattr(nn.Module, '__init__', lambda *_: pytest.fail('a module is made'))
    assert torch.equal(t(x), want)


@pytest.mark.parametrize('device', DEVICES)
def test_compiled_fused_models_are_one_graph(device):
    """(with torch's own run of the graph: the separate calls)"""
    tokens = torch.arange(16, device=device).view(2, 8)
    fused, separate = language_model(True, device), language_model(False, device)
    compiled = torch.compile(fused, backend='eager', fullgraph=True)
    assert torch.equal(compiled(tokens, return_loss=True), separate(tokens, return_loss=True))
    assert torch.equal(torch.compile(fused.transformer, backend='eager', fullgraph=True)(rows(device).bfloat16()), separate.transformer(rows(device).bfloat16()))


@pytest.mark.parametrize('fused', [False, True])
def test_a_read_out_of_another_kind_has_a_loss(fused):
    lm, tokens = language_model(fused, 'cpu'), torch.arange(16).view(2, 8)
    want = lm(tokens, return_loss=True)
    lm.to_logits = nn.Sequential(lm.to_logits)
    assert torch.equal(lm(tokens, return_loss=True), want)


@pytest.mark.parametrize('device', DEVICES)
def test_a_default_device_is_nobody_who_watches(device, monkeypatch):
    from simplicial_attention_amd import two_simplicial_transformer as module
    behind, fused, separate = [], stack(True, device), stack(False, device)
    x = rows(device)
    want = fused(x)
    monkeypatch.setattr(module, 'norm_behind', lambda *args, whole=module.norm_behind: behind.append(1) or whole(*args))
    with torch.device(device):
        assert torch.equal(fused(x), want)
        separate(x)
    assert len(behind) == 7


@pytest.mark.gpu
def test_a_default_device_leaves_the_kernels(monkeypatch):
    from simplicial_attention_amd import rms_norm
    from simplicial_attention_amd import two_simplicial_transformer as module
    called = []
    monkeypatch.setattr(rms_norm, 'add_rms_norm', lambda *args, kernel=rms_norm.add_rms_norm: called.append('norm') or kernel(*args))
    monkeypatch.setattr(module, 'linear_cross_entropy', lambda *args, kernel=module.linear_cross_entropy: called.append('loss') or kernel(*args))
    with torch.device('cuda'):
        language_model(True, 'cuda')(torch.arange(16, device='cuda').view(2, 8), return_loss=True)
    assert called == ['norm'] * 5 + ['loss']
